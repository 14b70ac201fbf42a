// Causal attention over packed sequences with f32 queries, at about f32 accuracy, on the 5th-generation tensor cores
// (sm_100a). 16-bit queries take attention_packed.cu, whose way of drawing units, fetching and guarding this follows.
//
// Queries and weights enter the MMA as sums of 16-bit terms of the keys' type: two f16 terms (22 bits) or three bf16
// terms (24 bits); each query row is first scaled by a power of two, and weights carry 2^14, so that the small terms
// stay normal f16 numbers. Every product so takes two or three MMAs, and one 128-row query tile keeps the tensor cores
// as busy as two of 16-bit queries: a unit of work is one query tile. Roles of a CTA's 12 warps:
//   0     draws units, issues the TMA loads of K and V tiles of 128 rows, in the order of their use
//   1     issues the MMAs: S = Q K^T into one of two score tiles, O = P V, P over the scores it came from (a third
//         term beside them)
//   2-3   guard the V tiles that the mask cuts
//   4-11  two threads a row, each half of the keys of a tile: the query's terms, softmax, weights, and half of O
// S(j + 1) is made while tile j's softmax runs. The MMA truncates its sums, and an O summed up in tensor memory over a
// long sequence would drift by a truncation a step, always towards zero: so O of each tile is a sum of its own, read
// back and added in f32 by the threads that hold O in registers, while the tensor cores work on the next tile.
//
// Bound by the tensor cores for long prompts: 4 (f16) or 6 (bf16) products of 128 x 128 x HD a tile, of 512 cycles each
// at HD 128 (20,545 tokens in prompts of up to 4096, 28 / 4 heads: 886 us with f16 keys, 1187 with bf16, 0.69 and 0.77 of
// their rate). By a unit's own chain for short ones (2563 tokens in prompts of up to 512: 53.5 us, 60.5 with bf16 keys).
#include <mutex>

#include "ops.cuh"
#include "packed.cuh"
#include "packed_attn.cuh"
#include "suite.h"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace l0b {

namespace {

constexpr int kUnitSlots = 4;  // drawn units in flight
constexpr int kThreads = 384;
constexpr int kRowThreads = 256;
constexpr float kWeightBits = 14.f;  // weights are at most 2^14

template <bool BF> constexpr int kTerms = BF ? 3 : 2;
template <bool BF> constexpr int kRing = BF ? 3 : 4;  // K and V tiles in shared memory, beside the query's terms

struct PackedF32Launch {
    CUtensorMap kmap, vmap;  // [rows, heads * hd], box {64, 128}
    PackedAttnParams a;
    unsigned* counters;      // [0] units drawn beyond each CTA's first, [1] CTAs done; zero at rest
};

// One unit, worked out by the drawing thread and handed on in shared memory.
struct Unit {
    PackedSeq s;
    int head, tok;  // query head, first row within the sequence
    int rows;       // live rows
    int nt;         // key tiles, -1: no more units
    int full;       // key tiles that every row sees whole

    // Places in the order of the fetched tiles: K_0, then K_(j + 1) and V_j in turn.
    __device__ __forceinline__ int k_entry(int j) const { return j == 0 ? 0 : 2 * j - 1; }
    __device__ __forceinline__ int v_entry(int j) const { return j + 1 < nt ? 2 * j + 2 : 2 * j + 1; }
};

__device__ __forceinline__ int units_of(const PackedAttnParams& a, int n) { return (n + kRows - 1) / kRows * a.nh; }

__device__ __forceinline__ Unit unit_at(const PackedAttnParams& a, const int* pre, int u) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= u) lo = mid;
        else hi = mid;
    }
    Unit x;
    x.s = packed_seq(a, lo);
    const int r = u - pre[lo], blocks = (pre[lo + 1] - pre[lo]) / a.nh;
    x.head = r % a.nh;
    x.tok = (blocks - 1 - r / a.nh) * kRows;  // late rows see the most keys: first
    x.rows = min(kRows, x.s.n - x.tok);
    const int first = x.s.m - x.s.n + x.tok, last = first + x.rows - 1;
    x.nt = last >= 0 ? last / kRows + 1 : 0;
    x.full = min(x.nt, max(0, first + 1) / kRows);
    return x;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    return DT<T>::id == L0B_F16 ? half2_bits_to_float2(w) : bf162_bits_to_float2(w);
}

// (a, b) as a sum of N pairs of 16-bit values.
template <typename T, int N>
__device__ __forceinline__ void split(float a, float b, uint32_t (&term)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        term[i] = pack2<T>(a, b);
        if (i + 1 < N) {
            const float2 f = unpack2<T>(term[i]);
            a -= f.x;
            b -= f.y;
        }
    }
}

template <bool BF, int HD>
__global__ void __launch_bounds__(kThreads, 1) packed_f32_kernel(const __grid_constant__ PackedF32Launch L) {
    using T = typename std::conditional<BF, __nv_bfloat16, __half>::type;
    constexpr int N = kTerms<BF>, R = kRing<BF>, BLOCKS = HD / 64, TILE = BLOCKS * kSub;
    constexpr uint32_t kIdescS = mma_idesc(BF, kRows, false), kIdescO = mma_idesc(BF, HD, true);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = smem;             // [N terms][TILE]
    uint8_t* kv_s = smem + N * TILE; // [R][TILE]
    // [8 row warps][32 rows of 64 bytes] of the epilogue; before it [tile & 1][half][row]: what a row's threads exchange
    uint8_t* stage_s = kv_s + R * TILE;
    int* pre = reinterpret_cast<int*>(stage_s + 8 * 2048);    // [count + 1] units before each sequence
    __shared__ __align__(8) uint64_t bars[1 + 3 * R + 2 * 2 + 3 + 2 * kUnitSlots];
    __shared__ Unit unit_s[kUnitSlots];
    __shared__ int scan_s[kThreads / 32], any_bad_s[8];
    __shared__ uint32_t bad_s[8][2][4];  // [unit & 7][cut tile]: value rows that are not finite
    __shared__ float factor_s[kRows];
    __shared__ uint32_t tmem_s;
    __shared__ int descends_s;
    const PackedAttnParams& a = L.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t q_full = smem_addr(bars), kv_full = q_full + 8, kv_empty = kv_full + 8 * R, v_ok = kv_empty + 8 * R;
    const uint32_t s_full = v_ok + 8 * R, p_ready = s_full + 16, o_full = p_ready + 16, o_free = o_full + 8;
    const uint32_t rows_bar = o_free + 8, drawn = rows_bar + 8, read = drawn + 8 * kUnitSlots;

    if (threadIdx.x == 0) {
        bar_init(q_full, kRowThreads);
        for (int i = 0; i < R; ++i) {
            bar_init(kv_full + 8 * i, 1);
            bar_init(kv_empty + 8 * i, 3);  // the MMAs and both guard warps
            bar_init(v_ok + 8 * i, 2);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(s_full + 8 * b, 1);
            bar_init(p_ready + 8 * b, kRowThreads);
        }
        bar_init(o_full, 1);
        bar_init(o_free, kRowThreads);
        bar_init(rows_bar, kRowThreads);
        for (int i = 0; i < kUnitSlots; ++i) {
            bar_init(drawn + 8 * i, 1);
            bar_init(read + 8 * i, 11);  // the MMA warp, two guard warps, eight row warps
        }
        bar_init_fence();
        descends_s = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.kmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.vmap)) : "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    tc_after();
    // Columns: scores and weight terms 0 and 1 of even and odd tiles, O, third terms of even and odd tiles.
    const uint32_t tmem = tmem_s, o_col = tmem + 2 * kRows, p2_col = tmem + 3 * kRows;

    const bool fine = packed_scan(a, pre, scan_s, &descends_s, [&](int n) { return units_of(a, n); });
    const int total = pre[a.count];
    bool ok = true;  // false once a bounded wait gave up: the role stops
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (ok) ok = bar_wait(bar, parity);
        return ok;
    };
    auto wait_warp = [&](uint32_t bar, uint32_t parity) {  // by a whole warp, which goes on or stops together
        if (ok) ok = bar_wait(bar, parity);
        return ok = __all_sync(0xffffffffu, ok);
    };
    int taken = 0;
    auto next_unit = [&](Unit& x) {  // false at the end
        const int slot = taken % kUnitSlots;
        if (!wait_warp(drawn + 8 * slot, (taken / kUnitSlots) & 1)) return false;
        x = unit_s[slot];
        __syncwarp();
        if (lane == 0) bar_arrive(read + 8 * slot);
        ++taken;
        return __shfl_sync(0xffffffffu, x.nt, 0) >= 0;
    };

    // The launch's 168 registers a thread are dealt anew: 88 for the first warpgroup, 208 for the row threads.
    // Query starts that descend: nothing runs.
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (!fine) {
    } else if (warp == 0) {
        if (lane == 0) {
            proxy_fence();
            int e = 0;
            int drawn_units = 0;
            // Draws, works out and hands on the next unit: one ahead of the unit whose tiles are being fetched.
            auto draw = [&]() {
                Unit x;
                unsigned u = blockIdx.x;
                if (drawn_units > 0) u = atomicAdd(L.counters, 1u) + gridDim.x;
                const int slot = drawn_units % kUnitSlots;
                if (u < static_cast<unsigned>(total)) x = unit_at(a, pre, static_cast<int>(u));
                else x.nt = -1;
                if (!wait(read + 8 * slot, ((drawn_units / kUnitSlots) & 1) ^ 1)) x.nt = -1;
                unit_s[slot] = x;
                any_bad_s[drawn_units & 7] = 0;
                bar_arrive(drawn + 8 * slot);
                ++drawn_units;
                return x;
            };
            Unit next = draw();
            while (next.nt >= 0 && ok) {
                const Unit x = next;
                if (x.nt == 0) next = draw();
                const int kvh = x.head / (a.nh / a.nkv);
                for (int k = 0; k < 2 * x.nt; ++k, ++e) {
                    const int st = e % R;
                    const bool is_v = k > 0 && (k == 2 * x.nt - 1 || (k & 1) == 0);
                    const int j = is_v ? (k == 2 * x.nt - 1 ? x.nt - 1 : (k - 2) >> 1) : (k + 1) >> 1;
                    if (!wait(kv_empty + 8 * st, ((e / R) & 1) ^ 1)) break;
                    bar_expect(kv_full + 8 * st, TILE);
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b)
                        tma_load(smem_addr(kv_s) + st * TILE + b * kSub, is_v ? &L.vmap : &L.kmap, kv_full + 8 * st,
                                 kvh * HD + 64 * b, x.s.k0 + j * kRows);
                    if (k == 0) next = draw();
                }
            }
            if (!ok) {  // no copy of this CTA's stays in flight behind it
                for (int i = max(0, e - R); i < e; ++i) bar_wait(kv_full + 8 * (i % R), (i / R) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        int e = 0, units = 0, made = 0, read_p = 0, outs = 0;  // fetched tiles before this unit; uses of each barrier
        uint32_t guarded = 0;                                  // phase bits of v_ok
        Unit x;
        while (next_unit(x)) {
            if (x.nt == 0) continue;
            if (!wait_warp(q_full, units++ & 1)) break;
            tc_after();
            auto scores = [&](int j) {  // S = Q K_j^T, small terms first
                const int n = e + x.k_entry(j), st = n % R, b = made & 1;
                if (!wait_warp(kv_full + 8 * st, (n / R) & 1)) return;
                tc_after();
                const uint32_t k = smem_addr(kv_s) + st * TILE;
#pragma unroll
                for (int t = N - 1; t >= 0; --t) {
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        const uint32_t at = (i >> 2) * kSub + (i & 3) * 32;
                        mma_ss(tmem + b * kRows, k_major_desc(smem_addr(q_s) + t * TILE + at), k_major_desc(k + at), kIdescS,
                               t < N - 1 || i > 0);
                    }
                }
                tc_commit(s_full + 8 * b);
                tc_commit(kv_empty + 8 * st);
                ++made;
            };
            scores(0);
            if (x.nt > 1) scores(1);
            for (int j = 0; j < x.nt && ok; ++j) {
                const int n = e + x.v_entry(j), st = n % R, b = read_p & 1;
                if (!wait_warp(kv_full + 8 * st, (n / R) & 1)) break;
                if (j >= x.full) {
                    if (!wait_warp(v_ok + 8 * st, (guarded >> st) & 1)) break;
                    guarded ^= 1u << st;
                }
                if (!wait_warp(o_free, (outs & 1) ^ 1)) break;
                if (!wait_warp(p_ready + 8 * b, (read_p >> 1) & 1)) break;
                tc_after();
                const uint32_t v = smem_addr(kv_s) + st * TILE;
#pragma unroll
                for (int t = N - 1; t >= 0; --t) {
                    const uint32_t p = t < 2 ? tmem + b * kRows + t * 64 : p2_col + b * 64;
#pragma unroll
                    for (int i = 0; i < kRows / 16; ++i)
                        mma_ts(o_col, p + i * 8, n_major_desc(v + i * 2048), kIdescO, t < N - 1 || i > 0);
                }
                tc_commit(o_full);
                tc_commit(kv_empty + 8 * st);
                ++outs;
                ++read_p;
                if (j + 2 < x.nt) scores(j + 2);
            }
            e += 2 * __shfl_sync(0xffffffffu, x.nt, 0);  // known to be uniform, and the stages with it
        }
        if (!ok) {  // MMAs in flight end before the tensor memory goes
            tc_commit(o_full);
            bar_wait(o_full, outs & 1);
        }
    } else {
        int e = 0;
        for (int i = 0;; ++i) {
            Unit x;
            if (!next_unit(x)) break;
            int j = 0;  // V tiles seen
            for (int k = 0; k < 2 * x.nt && ok; ++k, ++e) {
                const int st = e % R;
                // Every tile is waited for, so that the guard is never a round of the ring ahead or behind.
                if (!wait_warp(kv_full + 8 * st, (e / R) & 1)) break;
                const bool is_v = k > 0 && (k == 2 * x.nt - 1 || (k & 1) == 0);
                if (is_v && j >= x.full) {
                    uint32_t bad[2];
                    guard_rows<BF, BLOCKS>(kv_s + st * TILE, (warp - 2) * 64, x.s.m - j * kRows, lane, bad);
                    if (lane < 2) {
                        const uint32_t mine = lane ? bad[1] : bad[0];
                        bad_s[i & 7][(j - x.full) & 1][(warp - 2) * 2 + lane] = mine;
                        if (mine) any_bad_s[i & 7] = 1;
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) bar_arrive(v_ok + 8 * st);
                }
                if (lane == 0) bar_arrive(kv_empty + 8 * st);
                j += is_v;
            }
        }
    }
    } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    if (fine) {
        const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;  // keys 64 half .. + 63 of each tile, dims likewise
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        constexpr int DIMS = HD / 2;  // of O, a thread
        uint8_t* stage = stage_s + (warp - 4) * 2048;
        float(*swap)[2][kRows] = reinterpret_cast<float(*)[2][kRows]>(stage_s);
        int made = 0, outs = 0, syncs = 0;
        // All row threads; bounded, as every wait here. Weights go over scores that the row's other thread, in another
        // warp, has read: the fences order its tensor-memory loads before this thread's stores behind the barrier.
        auto rows_sync = [&]() {
            tc_before();
            bar_arrive(rows_bar);
            wait_warp(rows_bar, syncs++ & 1);
            tc_after();
        };
        // Query terms of a unit: a warp's 16 rows, eight rows' loads in flight, a row spread over the lanes. The scores
        // that read the last unit's terms are done: every row thread has seen its last.
        auto stage_query = [&](const Unit& x) {
            if (x.nt == 0) return;
            for (int r0 = 0; r0 < 16; r0 += 8) {
                float y[8][HD / 32];
                const int row0 = (warp - 4) * 16 + r0;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float* q = static_cast<const float*>(a.q) +
                                     static_cast<long long>(x.s.q0 + x.tok + min(row0 + r, x.rows - 1)) * a.q_stride +
                                     x.head * HD + lane * (HD / 32);
                    if constexpr (HD == 128) {
                        const float4 w = *reinterpret_cast<const float4*>(q);
                        y[r][0] = w.x; y[r][1] = w.y; y[r][2] = w.z; y[r][3] = w.w;
                    } else {
                        const float2 w = *reinterpret_cast<const float2*>(q);
                        y[r][0] = w.x; y[r][1] = w.y;
                    }
                }
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float top = 0.f;
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) top = fmaxf(top, fabsf(y[r][k]));
                    const int e = static_cast<int>(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127;
                    // 2^bits lifts the row's largest value to [2^13, 2^14); what is not finite stays so
                    const int bits = min(13 - e, 126);
                    const float up = __int_as_float((127 + bits) << 23);
                    if (lane == 0) factor_s[row0 + r] = a.scale * 1.44269504088896341f * __int_as_float((127 - bits) << 23);
                    uint32_t term[HD / 64][N];
#pragma unroll
                    for (int k = 0; k < HD / 64; ++k) split<T, N>(y[r][2 * k] * up, y[r][2 * k + 1] * up, term[k]);
                    const int d = lane * (HD / 32);  // first dim
#pragma unroll
                    for (int t = 0; t < N; ++t) {
                        uint8_t* at = q_s + t * TILE + (d >> 6) * kSub + (row0 + r) * 128 +
                                      ((((d & 63) >> 3) ^ ((row0 + r) & 7)) << 4) + (d & 7) * 2;
                        if constexpr (HD == 128) *reinterpret_cast<uint2*>(at) = make_uint2(term[0][t], term[HD / 64 - 1][t]);
                        else *reinterpret_cast<uint32_t*>(at) = term[0][t];
                    }
                }
            }
            proxy_fence();
            bar_arrive(q_full);
        };
        Unit x;
        bool have = next_unit(x);
        if (have) {
            stage_query(x);
            rows_sync();  // the rows' factors are there
        }
        for (int i = 0; have && ok; ++i) {
            const float f = factor_s[row];
            const int limit = x.s.m - x.s.n + x.tok + row;  // the last key this row sees
            float ref = kNegInf, sum = 0.f, keep = 1.f, o[DIMS];
#pragma unroll
            for (int k = 0; k < DIMS; ++k) o[k] = 0.f;
            auto take_out = [&]() {  // O of the tile before: o = o keep + O
                if (!wait_warp(o_full, outs++ & 1)) return;
                tc_after();
#pragma unroll
                for (int b = 0; b < DIMS / 32; ++b) {
                    uint32_t w[32];
                    tmem_load32(o_col + lanes + half * DIMS + 32 * b, w);
                    tmem_loaded(w);
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[32 * b + k] = fmaf(o[32 * b + k], keep, __uint_as_float(w[k]));
                }
                tc_before();
                bar_arrive(o_free);
            };
            for (int j = 0; j < x.nt; ++j) {
                const int b = made & 1;
                if (!wait_warp(s_full + 8 * b, (made >> 1) & 1)) break;
                ++made;
                tc_after();
                const uint32_t s_at = tmem + b * kRows + lanes;
                uint32_t s[2][32];
#pragma unroll
                for (int q = 0; q < 2; ++q) tmem_load32(s_at + 64 * half + 32 * q, s[q]);
#pragma unroll
                for (int q = 0; q < 2; ++q) tmem_loaded(s[q]);
                if (j >= x.full) {
                    const int last = limit - j * kRows - 64 * half;
#pragma unroll
                    for (int k = 0; k < 64; ++k)
                        if (k > last) s[k >> 5][k & 31] = __float_as_uint(kNegInf);
                }
                float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                for (int k = 0; k < 16; ++k) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) top[q] = fmaxf(top[q], __uint_as_float(s[q & 1][2 * k + (q >> 1)]));
                }
                const float mine = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                swap[j & 1][half][row] = mine;
                rows_sync();  // and both halves' scores are in registers: weights may go over them
                // In exp2's units; the scale is positive, so the largest stays the largest.
                const float now = fmaxf(ref, fmaxf(mine, swap[j & 1][half ^ 1][row]) * f);
                const float next_keep = now == ref ? 1.f : exp2_fast(ref - now);
                ref = now;
                const float shift = now == kNegInf ? 0.f : now - kWeightBits;
                float add[2] = {0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t w[N][16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float y0 = exp2_fast(fmaf(__uint_as_float(s[q][2 * k]), f, -shift));
                        const float y1 = exp2_fast(fmaf(__uint_as_float(s[q][2 * k + 1]), f, -shift));
                        add[0] += y0;
                        add[1] += y1;
                        uint32_t term[N];
                        split<T, N>(y0, y1, term);
#pragma unroll
                        for (int t = 0; t < N; ++t) w[t][k] = term[t];
                    }
#pragma unroll
                    for (int t = 0; t < N; ++t)
                        tmem_store16((t < 2 ? s_at + t * 64 : p2_col + lanes + b * 64) + 32 * half + 16 * q, w[t]);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_before();
                bar_arrive(p_ready + 8 * b);
                sum = fmaf(sum, next_keep, add[0] + add[1]);
                if (j > 0) take_out();
                keep = next_keep;
            }
            // The next unit's query terms before this one's end: its first scores are made meanwhile.
            Unit y;
            const bool more = ok && next_unit(y);
            if (more) stage_query(y);
            if (x.nt > 0 && ok) take_out();
            if (!ok) break;
            swap[0][half][row] = sum;
            rows_sync();
            const float all = swap[0][0][row] + swap[0][1][row], inv = limit < 0 ? 0.f : 1.f / all;
            rows_sync();  // the sums are read: their place is the epilogue's
            if (!ok) break;
            const bool any_bad = x.nt > 0 && *reinterpret_cast<volatile int*>(&any_bad_s[i & 7]) != 0;
            if (any_bad && row < x.rows) {
                // Values that the guard set aside, where this row sees them.
                for (int j = x.full; j < x.nt; ++j) {
                    for (int w = 0; w < 4; ++w) {
                        for (uint32_t bits = bad_s[i & 7][(j - x.full) & 1][w]; bits; bits &= bits - 1) {
                            const int key = j * kRows + w * 32 + __ffs(bits) - 1;
                            if (key > limit) break;
                            const float p = weight_anew<T, HD>(a, x.s, x.head, x.tok + row, key, a.scale * 1.44269504088896341f,
                                                               ref - kWeightBits);
                            const T* v = static_cast<const T*>(a.v) + static_cast<long long>(x.s.k0 + key) * a.v_stride +
                                         x.head / (a.nh / a.nkv) * HD + half * DIMS;
#pragma unroll
                            for (int k = 0; k < DIMS; ++k) o[k] = fmaf(p, load_as_float(v, DT<T>::id, k), o[k]);
                        }
                    }
                }
            }
            __syncwarp();
            // 32 rows of 64 bytes at a time through shared memory: four lanes store one row's 64 bytes.
            float* out = static_cast<float*>(a.out) + static_cast<long long>(x.s.q0 + x.tok + (warp & 3) * 32) * a.out_stride +
                         x.head * HD + half * DIMS;
#pragma unroll
            for (int b = 0; b < DIMS / 16; ++b) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<float4*>(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) =
                        make_float4(o[16 * b + 4 * k] * inv, o[16 * b + 4 * k + 1] * inv, o[16 * b + 4 * k + 2] * inv,
                                    o[16 * b + 4 * k + 3] * inv);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = k * 8 + (lane >> 2), piece = lane & 3;
                    const float4 w = *reinterpret_cast<const float4*>(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
                    if ((warp & 3) * 32 + r < x.rows) *reinterpret_cast<float4*>(out + r * a.out_stride + 16 * b + piece * 4) = w;
                }
                __syncwarp();
            }
            rows_sync();  // every warp is done with its stage: the next unit's exchanges may take the place
            have = more;
            if (more) x = y;
        }
    }
    }
    if (!ok && a.error) atomicOr(a.error, 1);
    tc_before();
    __syncthreads();
    if (warp == 0) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (threadIdx.x == 0 && fine) {
        __threadfence();
        if (atomicAdd(L.counters + 1, 1u) == gridDim.x - 1) {  // every CTA has drawn its last
            L.counters[0] = 0;
            L.counters[1] = 0;
        }
    }
}

template <bool BF, int HD>
l0b_status launch(l0b_suite* s, l0b_device* d, const PackedAttnParams& a) {
    auto kernel = packed_f32_kernel<BF, HD>;
    constexpr size_t tiles = 1024 + static_cast<size_t>(kTerms<BF> + kRing<BF>) * (HD / 64) * kSub + 8 * 2048;
    {
        static bool configured[64] = {};
        static std::mutex mu;
        std::lock_guard<std::mutex> lock(mu);
        if (d->index >= 64 || !configured[d->index]) {
            L0B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                static_cast<int>(tiles + 4 * (kMaxSequences + 1))));
            if (d->index < 64) configured[d->index] = true;
        }
    }
    PackedF32Launch L;
    std::memset(&L, 0, sizeof L);
    const auto type = BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const long long kvw = static_cast<long long>(a.nkv) * HD, kv_rows = a.kv_tokens > 0 ? a.kv_tokens : 1;
    L0B_TRY(tensor_map_2d(&L.kmap, type, 2, a.k, kvw, kv_rows, a.k_stride, 64, kRows, CU_TENSOR_MAP_SWIZZLE_128B));
    L0B_TRY(tensor_map_2d(&L.vmap, type, 2, a.v, kvw, kv_rows, a.v_stride, 64, kRows, CU_TENSOR_MAP_SWIZZLE_128B));
    L.a = a;
    L.counters = s->packed_counters;
    return d->launch(kernel, dim3(d->sm_count), dim3(kThreads), tiles + 4 * (static_cast<size_t>(a.count) + 1), L);
}

}  // namespace

l0b_status k_attention_packed_f32(l0b_suite* s, l0b_device* d, const PackedAttnParams& p) {
    if (p.kv_dtype == L0B_F16) return p.hd == 64 ? launch<false, 64>(s, d, p) : launch<false, 128>(s, d, p);
    return p.hd == 64 ? launch<true, 64>(s, d, p) : launch<true, 128>(s, d, p);
}

}  // namespace l0b
