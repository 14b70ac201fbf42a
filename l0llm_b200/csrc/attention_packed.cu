// Causal attention over packed sequences on the 5th-generation tensor cores (sm_100a): 16-bit queries. f32 queries
// take attention_packed_f32.cu.
//
// A unit of work is two tiles of 128 query rows of one sequence that read the same keys: two query heads of one KV
// head over the same rows where the group is even (PAIR), else two consecutive row blocks of one head. CTAs (one per
// SM) draw units from a counter: sequences in their order, each one's last rows, which see the most keys, first (16 prompts
// in ascending, descending and mixed order of length: 437 to 442 us). The kernel reads the sequences' starts on the
// device, so one launch serves any mix of lengths. Few rows behind a long prefix leave SMs without a unit: 1 to 128 rows
// behind 7994 keys take 110 us, whatever their number. Roles of a CTA's 12 warps:
//   0     draws units, issues the TMA loads: Q tiles, then K and V tiles of 128 rows through a ring of four stages
//   1     issues the MMAs: S_t = Q_t K^T and O_t += P_t V, S, P and O in tensor memory (S 128 columns a tile, P over
//         the S it came from, O HD columns), V read as it lies (N-major operand)
//   2-3   guard the V tiles that the mask cuts (below)
//   4-7   softmax of tile 0, a thread per row; 8-11 of tile 1
// While one tile's softmax runs the tensor cores work on the other tile. The softmax is online in exp2 with a lazy
// reference: O is rescaled only when a row's maximum has grown by 2^8, which after the first tiles is rare, and then
// by the row's own softmax thread: S(j) is issued behind O += P(j - 1) V(j - 1), so whoever has S(j) may touch O.
//
// Rows and keys of neighbouring sequences share the tiles' edges. Scores out of a row's sight are replaced, not
// added to, so nothing of K reaches it; but 0 * NaN is NaN in P V. So in a tile that some row sees only in part the
// guard zeroes value rows behind the sequence, and value rows that hold an infinity or a NaN, which it notes; the
// rows that do see such a key add its share in the epilogue.
//
// Probabilities are rounded once to the operands' type (its MMA takes no other), their sum is taken before that. f16
// weights carry a factor 2^7: with the 2^8 that the reference may lag behind, 2^15 is the largest power of two that f16
// holds, and half of its smallest step is then 2^-32 of the row's largest weight at most. (Without it 131,071 keys at 2^-26
// of one other's weight, 2^-9 of the result, were lost.)
//
// The MMA truncates, always towards zero: seen on values chosen for it, a step of 16 keys cuts each product at about 2^-25
// of the sum and the sum at 2^-23, so it costs 5 * 2^-23 of the sum at most. 131,072 keys alike in one sum came out 8.5e-4
// low, 1,048,576 keys 6.8e-3. So O is summed in tensor memory over 8192 keys at most (512 steps: 3.1e-4 at most, less than
// half a step of f16; 5e-5 for keys alike) and then added to a carry in f32, in global memory, since tensor memory is full
// and the registers are taken: 128 KB a CTA, written by the row's own thread and read back by it. One carry a row costs 16,384
// tokens 2% (4.10 -> 4.18 ms); over 16,384 keys at a time they would need none, but could lose more than f16's half step.
//
// The tensor cores and the exponentials have as much to do: 2 x 128 x 128 exponentials and four 128 x 128 x HD products
// take about 2048 cycles each at HD 128. A pair of tiles takes 3250: the MMA warp's waits and commits stand between the
// products. 16,384 tokens of 64 / 8 heads in bf16 take 4.18 ms, 1.05 PFLOP/s, at the power limit (SM clock 1.70 GHz).
// Measured and not kept, each in turn with the kept kernel in single launches on 17,495 tokens behind prefixes, 28 / 4 heads:
// an MMA warp for each query tile, whose products then interleave (14% slower), and two threads a row (13%).
#include <mutex>

#include "ops.cuh"
#include "packed.cuh"
#include "packed_attn.cuh"
#include "suite.h"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace l0b {

namespace {

constexpr int kRing = 4;       // K and V tiles in shared memory
constexpr int kUnitSlots = 4;  // drawn units in flight
constexpr int kThreads = 384;
template <bool BF> constexpr float kLiftBits = BF ? 0.f : 7.f;  // of the weights
constexpr int kCarryTiles = 64;  // key tiles that O is summed over in tensor memory

struct PackedLaunch {
    CUtensorMap qmap, kmap, vmap;  // [rows, heads * hd], box {64, 128}
    PackedAttnParams a;
    unsigned* counters;  // [0] units drawn beyond each CTA's first, [1] CTAs done; zero at rest
    float* carry;        // [CTA][query tile][dim / 4][row][4] sums of O
};

// One unit, worked out by the drawing thread and handed on in shared memory.
struct Unit {
    PackedSeq s;
    int head[2], tok[2];  // of each tile: query head, first row within the sequence
    int rows[2], nt[2];   // live rows, key tiles
    int full[2];          // key tiles that every row of the query tile sees whole
    int key_tiles;        // the larger nt, -1: no more units

    __device__ __forceinline__ bool cut(int j) const {  // some row sees key tile j in part
        return (j < nt[0] && j >= full[0]) || (j < nt[1] && j >= full[1]);
    }
    __device__ __forceinline__ int first_cut() const {
        const int c0 = nt[0] ? full[0] : key_tiles, c1 = nt[1] ? full[1] : key_tiles;
        return min(c0, c1);
    }
};

template <bool PAIR>
__device__ __forceinline__ int units_of(const PackedAttnParams& a, int n) {
    return PAIR ? (n + kRows - 1) / kRows * (a.nh / 2) : (n + 2 * kRows - 1) / (2 * kRows) * a.nh;
}

template <bool PAIR>
__device__ __forceinline__ Unit unit_at(const PackedAttnParams& a, const int* pre, int u) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= u) lo = mid;
        else hi = mid;
    }
    Unit x;
    x.s = packed_seq(a, lo);
    const int sets = PAIR ? a.nh / 2 : a.nh, r = u - pre[lo];
    const int blocks = (pre[lo + 1] - pre[lo]) / sets;
    const int block = blocks - 1 - r / sets, set = r % sets;  // late rows see the most keys: first
    x.head[0] = PAIR ? 2 * set : set;
    x.head[1] = PAIR ? 2 * set + 1 : set;
    x.tok[0] = block * (PAIR ? kRows : 2 * kRows);
    x.tok[1] = PAIR ? x.tok[0] : x.tok[0] + kRows;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        x.rows[t] = max(0, min(kRows, x.s.n - x.tok[t]));
        const int first = x.s.m - x.s.n + x.tok[t], last = first + x.rows[t] - 1;
        x.nt[t] = x.rows[t] > 0 && last >= 0 ? last / kRows + 1 : 0;
        x.full[t] = min(x.nt[t], max(0, first + 1) / kRows);
    }
    x.key_tiles = max(x.nt[0], x.nt[1]);
    return x;
}

template <bool BF, int HD, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) packed_tc_kernel(const __grid_constant__ PackedLaunch L) {
    using T = typename std::conditional<BF, __nv_bfloat16, __half>::type;
    constexpr int BLOCKS = HD / 64, TILE = BLOCKS * kSub;
    constexpr uint32_t kIdescS = mma_idesc(BF, kRows, false), kIdescO = mma_idesc(BF, HD, true);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = smem;               // [2][TILE]
    uint8_t* kv_s = smem + 2 * TILE;   // [kRing][TILE]
    uint8_t* stage_s = kv_s + kRing * TILE;  // [8 softmax warps][32 rows of 64 bytes] of the epilogue
    int* pre = reinterpret_cast<int*>(stage_s + 8 * 2048);  // [count + 1] units before each sequence
    __shared__ __align__(8) uint64_t bars[2 + 2 * kRing + 5 * 2 + kRing + 2 * kUnitSlots];
    __shared__ Unit unit_s[kUnitSlots];
    __shared__ int scan_s[kThreads / 32];
    // Value rows that are not finite: [unit & 7][cut tile & 3]. The roles are at most kUnitSlots units apart.
    __shared__ uint32_t bad_s[8][4][4];
    __shared__ int any_bad_s[8];
    __shared__ uint32_t tmem_s;
    __shared__ int descends_s;
    const PackedAttnParams& a = L.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t bar0 = smem_addr(bars);
    const uint32_t q_full = bar0, q_empty = bar0 + 8, kv_full = bar0 + 16, kv_empty = kv_full + 8 * kRing;
    const uint32_t s_full = kv_empty + 8 * kRing, p_ready = s_full + 16, o_full = p_ready + 32, o_empty = o_full + 16;
    const uint32_t v_ok = o_empty + 16, drawn = v_ok + 8 * kRing, read = drawn + 8 * kUnitSlots;

    if (threadIdx.x == 0) {
        bar_init(q_full, 1);
        bar_init(q_empty, 1);
        for (int i = 0; i < kRing; ++i) {
            bar_init(kv_full + 8 * i, 1);
            bar_init(kv_empty + 8 * i, i & 1 ? 3 : 1);  // V stages: the MMAs and both guard warps
            bar_init(v_ok + 8 * i, 2);
        }
        for (int t = 0; t < 2; ++t) {
            bar_init(s_full + 8 * t, 1);
            bar_init(p_ready + 16 * t, kRows);      // weights of keys 0-63 of a tile
            bar_init(p_ready + 16 * t + 8, kRows);  // of keys 64-127
            bar_init(o_full + 8 * t, 1);
            bar_init(o_empty + 8 * t, kRows);
        }
        for (int i = 0; i < kUnitSlots; ++i) {
            bar_init(drawn + 8 * i, 1);
            bar_init(read + 8 * i, 11);  // MMA thread, two guard warps, eight softmax warps
        }
        bar_init_fence();
        descends_s = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.qmap)) : "memory");
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
    const uint32_t tmem = tmem_s;

    const bool fine = packed_scan(a, pre, scan_s, &descends_s, [&](int n) { return units_of<PAIR>(a, n); });
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
    // The next drawn unit; false at the end.
    int taken = 0;
    auto next_unit = [&](Unit& x) {
        const int slot = taken % kUnitSlots;
        if (!wait_warp(drawn + 8 * slot, (taken / kUnitSlots) & 1)) return false;
        x = unit_s[slot];
        __syncwarp();
        if (lane == 0) bar_arrive(read + 8 * slot);
        ++taken;
        return __shfl_sync(0xffffffffu, x.key_tiles, 0) >= 0;
    };

    // The launch's 168 registers a thread are dealt anew: 88 for the first warpgroup, 208 for the softmax threads.
    // Query starts that descend: nothing runs.
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (!fine) {
    } else if (warp == 0) {
        if (lane == 0) {
            proxy_fence();
            int e = 0, q_uses = 0;
            int drawn_units = 0;
            // Draws, works out and hands on the next unit: one ahead of the unit whose tiles are being fetched.
            auto draw = [&]() {
                Unit x;
                unsigned u = blockIdx.x;
                if (drawn_units > 0) u = atomicAdd(L.counters, 1u) + gridDim.x;
                const int slot = drawn_units % kUnitSlots;
                if (u < static_cast<unsigned>(total)) x = unit_at<PAIR>(a, pre, static_cast<int>(u));
                else x.key_tiles = -1;
                if (!wait(read + 8 * slot, ((drawn_units / kUnitSlots) & 1) ^ 1)) x.key_tiles = -1;
                unit_s[slot] = x;
                any_bad_s[drawn_units & 7] = 0;
                bar_arrive(drawn + 8 * slot);
                ++drawn_units;
                return x;
            };
            Unit next = draw();
            while (next.key_tiles >= 0 && ok) {
                const Unit x = next;
                if (x.key_tiles == 0) next = draw();
                const int kvh = x.head[0] / (a.nh / a.nkv);
                for (int k = 0; k < 2 * x.key_tiles; ++k, ++e) {  // K_0, Q, V_0, K_1, V_1, ...
                    const int st = e % kRing;
                    if (!wait(kv_empty + 8 * st, ((e / kRing) & 1) ^ 1)) break;
                    bar_expect(kv_full + 8 * st, TILE);
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b)
                        tma_load(smem_addr(kv_s) + st * TILE + b * kSub, k & 1 ? &L.vmap : &L.kmap, kv_full + 8 * st,
                                 kvh * HD + 64 * b, x.s.k0 + (k >> 1) * kRows);
                    if (k > 0) continue;
                    if (!wait(q_empty, (q_uses & 1) ^ 1)) break;
                    ++q_uses;
                    bar_expect(q_full, ((x.nt[0] > 0) + (x.nt[1] > 0)) * TILE);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (x.nt[t] == 0) continue;
#pragma unroll
                        for (int b = 0; b < BLOCKS; ++b)
                            tma_load(smem_addr(q_s) + t * TILE + b * kSub, &L.qmap, q_full, x.head[t] * HD + 64 * b, x.s.q0 + x.tok[t]);
                    }
                    next = draw();
                }
            }
            if (!ok) {  // no copy of this CTA's stays in flight behind it
                if (q_uses > 0) bar_wait(q_full, (q_uses - 1) & 1);
                for (int i = max(0, e - kRing); i < e; ++i) bar_wait(kv_full + 8 * (i % kRing), (i / kRing) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        int e = 0, q_uses = 0;
        uint32_t p_uses[2] = {0, 0}, o_uses[2] = {0, 0}, guarded[kRing / 2] = {0, 0};  // V takes the odd stages
        Unit x;
        while (next_unit(x)) {
            if (x.key_tiles == 0) continue;
            if (!wait_warp(q_full, q_uses & 1)) break;
            ++q_uses;
            auto scores = [&](int t, int j) {  // S_t = Q_t K_j^T
                const int st = (e + 2 * j) % kRing;
                if (!wait_warp(kv_full + 8 * st, ((e + 2 * j) / kRing) & 1)) return;
                tc_after();
                const uint32_t q = smem_addr(q_s) + t * TILE, k = smem_addr(kv_s) + st * TILE;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                    const uint32_t at = (i >> 2) * kSub + (i & 3) * 32;
                    mma_ss(tmem + t * kRows, k_major_desc(q + at), k_major_desc(k + at), kIdescS, i > 0);
                }
                tc_commit(s_full + 8 * t);
                if (t == (j < x.nt[1] ? 1 : 0)) {  // the last tile that reads K_j
                    tc_commit(kv_empty + 8 * st);
                    if (j == x.key_tiles - 1) tc_commit(q_empty);
                }
            };
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (x.nt[t] > 0) scores(t, 0);
            for (int j = 0; j < x.key_tiles && ok; ++j) {
                bool have_v = false;
                const int st = (e + 2 * j + 1) % kRing;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (j >= x.nt[t] || !ok) continue;
                    if (!have_v) {
                        if (!wait_warp(kv_full + 8 * st, ((e + 2 * j + 1) / kRing) & 1)) break;
                        if (x.cut(j) && !wait_warp(v_ok + 8 * st, guarded[st >> 1]++ & 1)) break;
                        have_v = true;
                    }
                    if (j == 0 && !wait_warp(o_empty + 8 * t, (o_uses[t]++ & 1) ^ 1)) break;
                    const uint32_t v = smem_addr(kv_s) + st * TILE;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!wait_warp(p_ready + 16 * t + 8 * h, p_uses[t] & 1)) break;
                        tc_after();
#pragma unroll
                        for (int i = 4 * h; i < 4 * h + 4; ++i)
                            mma_ts(tmem + 2 * kRows + t * HD, tmem + t * kRows + i * 8, n_major_desc(v + i * 2048), kIdescO,
                                   j % kCarryTiles > 0 || i > 0);
                    }
                    ++p_uses[t];
                    if (t == (j < x.nt[1] ? 1 : 0)) tc_commit(kv_empty + 8 * st);
                    if (j + 1 < x.nt[t]) scores(t, j + 1);
                    else tc_commit(o_full + 8 * t);
                }
            }
            e += 2 * __shfl_sync(0xffffffffu, x.key_tiles, 0);  // known to be uniform, and the stages with it
        }
        if (!ok) {
            tc_commit(q_empty);  // MMAs in flight end before the tensor memory goes
            bar_wait(q_empty, (q_uses - 1) & 1);
        }
    } else {
        int e = 0;
        for (int i = 0;; ++i) {
            Unit x;
            if (!next_unit(x)) break;
            int nth = 0;
            for (int j = 0; j < x.key_tiles && ok; ++j) {
                // Every V tile is waited for, so that the guard is never a round of the ring ahead or behind.
                const int st = (e + 2 * j + 1) % kRing;
                if (!wait_warp(kv_full + 8 * st, ((e + 2 * j + 1) / kRing) & 1)) break;
                if (!x.cut(j)) {
                    if (lane == 0) bar_arrive(kv_empty + 8 * st);
                    continue;
                }
                uint8_t* v = kv_s + st * TILE;
                uint32_t bad[2];
                guard_rows<BF, BLOCKS>(v, (warp - 2) * 64, x.s.m - j * kRows, lane, bad);
                if (lane < 2) {
                    const uint32_t mine = lane ? bad[1] : bad[0];
                    bad_s[i & 7][nth & 3][(warp - 2) * 2 + lane] = mine;
                    if (mine) any_bad_s[i & 7] = 1;
                }
                ++nth;
                proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    bar_arrive(v_ok + 8 * st);
                    bar_arrive(kv_empty + 8 * st);
                }
            }
            e += 2 * x.key_tiles;
        }
    }
    } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    if (fine) {
        const int t = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + t * kRows + lanes, o_at = tmem + 2 * kRows + t * HD + lanes;
        const float c = a.scale * 1.44269504088896341f;
        uint8_t* stage = stage_s + (warp - 4) * 2048;
        float* carry = L.carry + (static_cast<size_t>(blockIdx.x) * 2 + t) * 128 * kRows + row * 4;
        uint32_t s_uses = 0, o_uses = 0;
        for (int i = 0;; ++i) {
            Unit x;
            if (!next_unit(x)) break;
            const int nt = x.nt[t], limit = x.s.m - x.s.n + x.tok[t] + row;  // the last key this row sees
            float ref = kNegInf, sum = 0.f;  // weights are exp2((s - ref) c + kLiftBits)
            auto shift_of = [&]() { return ref == kNegInf ? 0.f : fmaf(ref, c, -kLiftBits<BF>); };
            float carry_ref = kNegInf;       // the reference that the carry was last written under
            auto carry_scale = [&]() { return carry_ref == ref ? 1.f : exp2_fast((carry_ref - ref) * c); };
            for (int j = 0; j < nt; ++j) {
                if (!wait_warp(s_full + 8 * t, s_uses++ & 1)) break;
                tc_after();
                const bool anew = j % kCarryTiles == 0;  // O starts anew with this tile
                if (anew && j > 0) {
                    const float f = carry_scale();
#pragma unroll 1
                    for (int b = 0; b < HD / 32; ++b) {
                        uint32_t o[32];
                        tmem_load32(o_at + 32 * b, o);
                        tmem_loaded(o);
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            float4* at = reinterpret_cast<float4*>(carry + (32 * b + k) * kRows);
                            float4 w = make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]),
                                                   __uint_as_float(o[k + 3]));
                            if (j > kCarryTiles) {
                                const float4 was = *at;
                                w = make_float4(fmaf(was.x, f, w.x), fmaf(was.y, f, w.y), fmaf(was.z, f, w.z), fmaf(was.w, f, w.w));
                            }
                            *at = w;
                        }
                    }
                    carry_ref = ref;
                }
                uint32_t s[4][32];
#pragma unroll
                for (int b = 0; b < 4; ++b) tmem_load32(s_at + 32 * b, s[b]);
#pragma unroll
                for (int b = 0; b < 4; ++b) tmem_loaded(s[b]);
                if (j >= x.full[t]) {
                    const int last = limit - j * kRows;
#pragma unroll
                    for (int k = 0; k < 128; ++k)
                        if (k > last) s[k >> 5][k & 31] = __float_as_uint(kNegInf);
                }
                float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
#pragma unroll
                    for (int b = 0; b < 4; ++b) top[b] = fmaxf(fmaxf(top[b], __uint_as_float(s[b][k])), __uint_as_float(s[b][k + 1]));
                }
                const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                // The reference moves when it must: at the first keys seen, or when weights would pass 2^8 of it.
                const bool move = most > ref && !((most - ref) * c <= 8.f);
                if (__any_sync(0xffffffffu, move)) {
                    const float by = move ? exp2_fast((ref - most) * c) : 1.f;
                    if (!anew) {
#pragma unroll 1
                        for (int b = 0; b < HD / 32; ++b) {
                            uint32_t o[32];
                            tmem_load32(o_at + 32 * b, o);
                            tmem_loaded(o);
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * by);
                            tmem_store32(o_at + 32 * b, o);
                        }
                    }
                    if (move) {
                        ref = most;
                        sum *= by;
                    }
                }
                __syncwarp();
                const float shift = shift_of();
                const float2 c2 = make_float2(c, c), shift2 = make_float2(-shift, -shift);
                float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 y = ffma2(make_float2(__uint_as_float(s[b][2 * k]), __uint_as_float(s[b][2 * k + 1])), c2, shift2);
                        y.x = exp2_fast(y.x);
                        y.y = exp2_fast(y.y);
                        add[k & 1] = fadd2(add[k & 1], y);
                        w[k] = pack2<T>(y.x, y.y);
                    }
                    tmem_store16(s_at + 16 * b, w);
                    if (b & 1) {
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        tc_before();
                        bar_arrive(p_ready + 16 * t + 4 * (b - 1));
                    }
                }
                sum += (add[0].x + add[0].y) + (add[1].x + add[1].y);
            }
            if (x.rows[t] == 0 || !ok) continue;
            if (nt > 0) {
                if (!wait_warp(o_full + 8 * t, o_uses++ & 1)) break;
                tc_after();
            }
            // A row without keys gives zeros; one whose every score is -inf has no weights, and 0 / 0 says so.
            const float inv = limit < 0 ? 0.f : 1.f / sum;
            const bool any_bad = nt > 0 && *reinterpret_cast<volatile int*>(&any_bad_s[i & 7]) != 0;
            T* out = static_cast<T*>(a.out) + static_cast<long long>(x.s.q0 + x.tok[t] + (warp & 3) * 32) * a.out_stride + x.head[t] * HD;
#pragma unroll 1
            for (int b = 0; b < HD / 32; ++b) {
                uint32_t o[32];
                if (nt > 0) {
                    tmem_load32(o_at + 32 * b, o);
                    tmem_loaded(o);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = 0;
                }
                if (b == HD / 32 - 1 && nt > 0) {
                    tc_before();
                    bar_arrive(o_empty + 8 * t);
                }
                if (nt > kCarryTiles) {
                    const float f = carry_scale();
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const float4 was = *reinterpret_cast<const float4*>(carry + (32 * b + k) * kRows);
                        o[k] = __float_as_uint(fmaf(was.x, f, __uint_as_float(o[k])));
                        o[k + 1] = __float_as_uint(fmaf(was.y, f, __uint_as_float(o[k + 1])));
                        o[k + 2] = __float_as_uint(fmaf(was.z, f, __uint_as_float(o[k + 2])));
                        o[k + 3] = __float_as_uint(fmaf(was.w, f, __uint_as_float(o[k + 3])));
                    }
                }
                if (row < x.rows[t]) {
                    // Values that the guard set aside, where this row sees them.
                    int nth = 0;
                    for (int j = any_bad ? x.first_cut() : x.key_tiles; j < x.key_tiles; ++j) {
                        if (!x.cut(j)) continue;
                        for (int w = 0; w < 4; ++w) {
                            for (uint32_t bits = bad_s[i & 7][nth & 3][w]; bits; bits &= bits - 1) {
                                const int key = j * kRows + w * 32 + __ffs(bits) - 1;
                                if (key > limit) break;
                                const float f = weight_anew<T, HD>(a, x.s, x.head[t], x.tok[t] + row, key, c, shift_of());
                                const T* v = static_cast<const T*>(a.v) + static_cast<long long>(x.s.k0 + key) * a.v_stride +
                                             x.head[t] / (a.nh / a.nkv) * HD + 32 * b;
#pragma unroll
                                for (int k = 0; k < 32; ++k)
                                    o[k] = __float_as_uint(fmaf(f, load_as_float(v, DT<T>::id, k), __uint_as_float(o[k])));
                            }
                        }
                        ++nth;
                    }
                }
                // 32 rows of 64 bytes through shared memory, so that four lanes store one row's 64 bytes: a store of
                // 16 bytes of 32 rows takes 32 turns of the memory pipe, one of 64 bytes of 8 rows takes 8.
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint4 w;
                    w.x = pack2<T>(__uint_as_float(o[8 * k]) * inv, __uint_as_float(o[8 * k + 1]) * inv);
                    w.y = pack2<T>(__uint_as_float(o[8 * k + 2]) * inv, __uint_as_float(o[8 * k + 3]) * inv);
                    w.z = pack2<T>(__uint_as_float(o[8 * k + 4]) * inv, __uint_as_float(o[8 * k + 5]) * inv);
                    w.w = pack2<T>(__uint_as_float(o[8 * k + 6]) * inv, __uint_as_float(o[8 * k + 7]) * inv);
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = w;
                }
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = k * 8 + (lane >> 2), piece = lane & 3;
                    const uint4 w = *reinterpret_cast<const uint4*>(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
                    if ((warp & 3) * 32 + r < x.rows[t])
                        *reinterpret_cast<uint4*>(out + r * a.out_stride + 32 * b + piece * 8) = w;
                }
                __syncwarp();
            }
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

template <bool BF, int HD, bool PAIR>
l0b_status launch_tc(l0b_suite* s, l0b_device* d, const PackedAttnParams& a) {
    auto kernel = packed_tc_kernel<BF, HD, PAIR>;
    constexpr size_t tiles = 1024 + static_cast<size_t>(2 + kRing) * (HD / 64) * kSub + 8 * 2048;
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
    PackedLaunch L;
    std::memset(&L, 0, sizeof L);
    const auto type = BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const long long kvw = static_cast<long long>(a.nkv) * HD, kv_rows = a.kv_tokens > 0 ? a.kv_tokens : 1;
    L0B_TRY(tensor_map_2d(&L.qmap, type, 2, a.q, static_cast<long long>(a.nh) * HD, a.tokens, a.q_stride, 64, kRows,
                          CU_TENSOR_MAP_SWIZZLE_128B));
    L0B_TRY(tensor_map_2d(&L.kmap, type, 2, a.k, kvw, kv_rows, a.k_stride, 64, kRows, CU_TENSOR_MAP_SWIZZLE_128B));
    L0B_TRY(tensor_map_2d(&L.vmap, type, 2, a.v, kvw, kv_rows, a.v_stride, 64, kRows, CU_TENSOR_MAP_SWIZZLE_128B));
    L.a = a;
    L.counters = s->packed_counters;
    L.carry = s->packed_carry;
    return d->launch(kernel, dim3(d->sm_count), dim3(kThreads), tiles + 4 * (static_cast<size_t>(a.count) + 1), L);
}

template <bool BF>
l0b_status launch_as(l0b_suite* s, l0b_device* d, const PackedAttnParams& a) {
    // Two heads that share keys need no second row block, which the last rows of a sequence may not have. Pairs against
    // row blocks of one head, 32 / 8 heads of 128, bf16: 16 prompts of up to 2048 behind prefixes 465 and 490 us, 8 prompts
    // of up to 512 38 and 36 (head dim 64: 33 and 37).
    const bool pair = (a.nh / a.nkv) % 2 == 0;
    if (a.hd == 64) return pair ? launch_tc<BF, 64, true>(s, d, a) : launch_tc<BF, 64, false>(s, d, a);
    return pair ? launch_tc<BF, 128, true>(s, d, a) : launch_tc<BF, 128, false>(s, d, a);
}

}  // namespace

l0b_status k_attention_packed(l0b_suite* s, l0b_device* d, const PackedAttnParams& p) {
    // Units are counted in 32 bits: blocks of rows times heads.
    L0B_REQUIRE((static_cast<long long>(p.tokens) / kRows + p.count) * p.nh <= INT32_MAX, L0B_ERR_OUT_OF_RANGE,
                "%d rows of %d heads are too many for one call", p.tokens, p.nh);
    if (p.q_dtype == L0B_F32) return k_attention_packed_f32(s, d, p);
    return p.kv_dtype == L0B_BF16 ? launch_as<true>(s, d, p) : launch_as<false>(s, d, p);
}

}  // namespace l0b
