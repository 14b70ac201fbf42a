// Attention over the int8 KV cache (sm_100a, mma.sync m16n8k16 with f32 accumulators, TMA-fed).
//
// The work is flat: for every (sequence, group of query columns) -- an item -- its tiles of 4 KB of keys and 4 KB of
// values (32 slots of head dim 128, 64 of 64), in order: one list, the same for every KV head. A group of teams of
// warps, one team per head, takes an equal run of that list, whatever the mix of lengths, which the kernel reads on
// the device; one launch, one CTA per SM. So the teams that run side by side read the heads of the same slots, whole
// cache rows, at the same time: with each head's list split on its own (hd bytes out of every row) the DRAM pages
// were opened once per head, and 1.05 GB of 8 heads took 1.6 times as long as the same bytes of one head. A run
// crosses items: the part of it inside one item is a segment. A warp takes every TEAM-th tile of its team's segment,
// fetched by its own TMA two tiles ahead, segments ahead included, so HBM stays busy through their ends.
//
// The query columns of an item are the rows that share its keys (the heads of a group, times the tokens): the MMA's
// n = 8 (NT tiles of it). Keys are its m: S^T[16 slots, 8 columns] = K Q^T on the integer MMA, the codes as they lie
// in the cache and each query column as base-256 digits of its values, scaled by a power of two to 31 bits (bf16: 23)
// of the column's largest: exact sums and no conversion (turning keys to f16 took 160 of 790 instructions a tile).
// O^T[16 dims, 8] += V^T P^T takes the codes as f16, exactly (byte b ^ 0x80 under the exponent of 1024, minus 1152),
// and P^T in hi + lo f16 terms made from the scores' own registers by movmatrix; digits there would cost more than
// they save, since every output would have to be converted for every tile. No product is padded to 16 query rows,
// and nothing but the raw codes crosses shared memory. A block's key scale multiplies the scores; its value scale
// the product of its 32 slots, summed in f32 outside the MMA, which truncates its sums: 32 slots a sum keep that
// below the f32 rounding of the rest.
// Softmax online, per warp and column, in exp2; weights carry a factor 2^14 that keeps their lo terms normal f16.
//
// At a segment's end the team's warps meet in shared memory (each in the ring stage it has just read). An item that
// several groups share has its parts joined, in group order, by the team that arrives last (a counter per first team,
// which the joining team resets), so results do not depend on the order of arrival.
//
// Bound by latency between dependent instructions: at 142,126 slots of 8 heads of 128 half of the issue slots and half of
// the DRAM rate are used, and 12 warps fill the registers. 514,036 slots take 218 us, 4.8 TB/s; 41,159 slots of 4 heads
// 29.5 us, three tiles a warp.
#include <mutex>

#include "ops.cuh"
#include "packed.cuh"
#include "suite.h"
#include "tma.cuh"

namespace l0b {

namespace {

constexpr int kTileBytes = 4096;  // of keys, and of values
constexpr int kStages = 2;        // ring stages of a warp
constexpr float kWeightBits = 14.f;  // weights are at most 2^14 (f16 holds 2^16)

__host__ __device__ constexpr int warps_of(int NT) { return NT == 1 ? 12 : 8; }  // registers of two column tiles

struct Q8Launch {
    CUtensorMap kmap, vmap;  // codes as [count * max_seq, nkv * hd] bytes, box {hd, tile slots}
    AttnQ8Params a;
    float* part;             // [2 N][8 NT][hd] unnormalised sums of shared items' parts
    float* part_ml;          // [2 N][8 NT][2] their maxima and weight sums
    unsigned* counters;      // [N] arrivals, by the item's first team; zero at rest
};

// What a warp needs to know of one item, and the walk over items.
// An item takes kItemUnits units and one for each of its tiles: starting and ending one costs as much as some twenty
// tiles (query digits, the joining of states; 4 us of latency), and runs of equal length would be uneven without it.
// With 0, 10, 20 and 40 units, 28 / 4 heads of 128, f32, in us: 16 sequences of up to 4096 slots 38, 31, 30, 28; 64 of up
// to 1024 40, 32, 32, 33; 4 of up to 4096 25, 20, 19, 20; 64 of up to 16,384 169, 163, 159, 154.
constexpr int kItemUnits = 20;

struct Item {
    int seq, cg;       // sequence, column group
    int cgroups;       // column groups of the sequence
    int tiles;
    int len, n, row0;  // slots held, query rows, first packed row
    int base;          // unit of the first tile
};

template <int NT>
struct Walk {
    const AttnQ8Params& a;
    const int* pre;  // units before each sequence
    int slots;  // per tile

    __device__ __forceinline__ void sequence(int i, int& row0, int& n, int& len) const {
        const int s = a.starts ? a.starts[i] : i, e = a.starts ? a.starts[i + 1] : i + 1;
        row0 = clamp_start(s, a.tokens);
        n = max(0, clamp_start(e, a.tokens) - row0);
        len = max(0, min(a.lengths[i], a.max_seq));
    }
    __device__ __forceinline__ int column_groups(int n) const { return (n * (a.nh / a.nkv) + 8 * NT - 1) / (8 * NT); }
    __device__ __forceinline__ int tiles_of(int len) const { return max(1, (len + slots - 1) / slots); }
    __device__ __forceinline__ void load_sequence(Item& it) const {
        sequence(it.seq, it.row0, it.n, it.len);
        it.cgroups = column_groups(it.n);
        it.tiles = tiles_of(it.len);
    }
    // Units of a sequence of n rows and len slots.
    __device__ __forceinline__ int units(int n, int len) const { return column_groups(n) * (kItemUnits + tiles_of(len)); }
    // The item that holds unit u.
    __device__ __forceinline__ Item find(int u) const {
        int lo = 0, hi = a.count;  // pre[lo] <= u < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= u) lo = mid;
            else hi = mid;
        }
        Item it;
        it.seq = lo;
        load_sequence(it);
        it.cg = (u - pre[lo]) / (kItemUnits + it.tiles);
        it.base = pre[lo] + it.cg * (kItemUnits + it.tiles) + kItemUnits;
        return it;
    }
    __device__ __forceinline__ void next(Item& it) const {
        it.base += it.tiles + kItemUnits;
        if (++it.cg < it.cgroups) return;
        it.cg = 0;
        do ++it.seq;
        while (it.seq + 1 < a.count && pre[it.seq] == pre[it.seq + 1]);
        if (it.seq < a.count) load_sequence(it);
    }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Byte k of each of four words, side by side.
__device__ __forceinline__ uint32_t byte_of(const int (&x)[4], int k) {
    const uint32_t lo = __byte_perm(x[0], x[1], k | ((4 + k) << 4)), hi = __byte_perm(x[2], x[3], k | ((4 + k) << 4));
    return __byte_perm(lo, hi, 0x5410);
}

// Bytes (0, 1) and (2, 3) of u (codes ^ 0x80) as f16 pairs, exactly.
__device__ __forceinline__ uint32_t codes_f16(uint32_t u, uint32_t selector) {
    const uint32_t h = __byte_perm(u, 0x64646464u, selector);  // 1024 + u
    const uint32_t bias = 0x64806480u;                         // 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void team_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Weights enter the MMA as hi + lo f16 terms, but for bf16 results: next to their rounding (2^-9 relative) that of a
// weight to f16 (2^-12) is not seen, and 60 instructions a tile fall away.
template <typename T>
constexpr bool kWeightPairs = DT<T>::id != L0B_BF16;
// Digits of a query value. What they drop is relative to the column's LARGEST value (2^-30 of it at most with four, 2^-22
// with three), so a loud channel costs the others bits: beside one of 1e4 three digits were off by 1e-4 of the largest
// output, 19 times the bound of f32 sums. Four keep every bit of values down to 2^-7 of the largest, f16's down to 2^-19.
// Three hold a bf16 value's 8 bits down to 2^-14 of the largest. The fourth costs 6% (41,159 slots of 4 heads 27.9 -> 29.5
// us in f32, 514,036 of 8 heads 220 -> 237 us in bf16).
template <typename T>
constexpr int kDigits = DT<T>::id == L0B_BF16 ? 3 : 4;

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(warps_of(NT) * 32, 1) attn_q8_kernel(const __grid_constant__ Q8Launch L) {
    constexpr int W = warps_of(NT), COLS = 8 * NT;
    constexpr int SLOTS = kTileBytes / HD, MT = SLOTS / 16, HALVES = SLOTS / 32;
    constexpr int KS = HD / 32;   // 32-deep steps of K Q^T
    constexpr int DT_ = HD / 16;  // 16-dim tiles of O
    constexpr int ND = kDigits<T>, kTopBit = ND == 4 ? 30 : 22, kBias = ND == 4 ? 0x808080 : 0x8080;
    constexpr bool PAIRS = kWeightPairs<T>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int* pre = reinterpret_cast<int*>(ring + W * kStages * 2 * kTileBytes);
    __shared__ __align__(8) uint64_t bars[W * kStages * 2];  // keys, values of each stage
    __shared__ float ml_s[W][COLS][2];
    __shared__ int scan_s[W][2];
    __shared__ unsigned last_s[W];
    const AttnQ8Params& a = L.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Walk<NT> walk{a, pre, SLOTS};

    if (threadIdx.x == 0) {
        for (int i = 0; i < W * kStages * 2; ++i) bar_init(smem_addr(&bars[i]), 1);
        bar_init_fence();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.kmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.vmap)) : "memory");
    }
    pdl_wait();
    pdl_launch_dependents();

    // pre[i] = units before sequence i: every CTA scans the lengths (a few loads a thread).
    {
        const int per = (a.count + W * 32 - 1) / (W * 32), i0 = threadIdx.x * per, i1 = min(a.count, i0 + per);
        int units = 0, items = 0;
        bool descends = false;  // sequences could then share rows of out, which no order of writing settles
        for (int i = i0; i < i1; ++i) {
            int row0, n, len;
            walk.sequence(i, row0, n, len);
            descends |= a.starts && a.starts[i] > a.starts[i + 1];
            if (blockIdx.x == 0 && (descends || a.lengths[i] != len ||
                                    (a.starts && (a.starts[i] < 0 || a.starts[i + 1] > a.tokens))))
                flag_bad_index(a.error);
            units += walk.units(n, len);
            items += walk.column_groups(n);
        }
        int sum = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        items = __reduce_add_sync(0xffffffffu, items);
        __syncthreads();
        if (lane == 31) {
            scan_s[warp][0] = sum;
            scan_s[warp][1] = items;
        }
        if (__syncthreads_or(descends)) return;  // nothing runs
        int before = sum - units;
        for (int w = 0; w < warp; ++w) before += scan_s[w][0];
        for (int i = i0; i < i1; ++i) {
            int row0, n, len;
            walk.sequence(i, row0, n, len);
            pre[i] = before;
            before += walk.units(n, len);
        }
        if (threadIdx.x == 0) {
            int all = 0;
            for (int w = 0; w < W; ++w) all += scan_s[w][0];
            pre[a.count] = all;
        }
        __syncthreads();
    }
    const int U = pre[a.count];
    if (U == 0) return;
    // Long items: the CTA's warps share one run, which has the fewest parts to join. Short items (fewer tiles than
    // two rounds of the CTA's warps): teams of four, so that more items are worked on at once. All warps against four, 28 / 4
    // heads of 128, f32, in us: one sequence of 32,768 slots 27 and 53; 4 of up to 4096 19 and 28; 16 of up to 4096 29 and
    // 29; 64 of up to 512 29 and 24. The rule looks at tiles alone: many long items would gain 5% from four (64 of up to
    // 16,384: 151 and 143), 4 of up to 512 lose 3 us to them (13 and 16).
    int items = 0;
    for (int w = 0; w < W; ++w) items += scan_s[w][1];
    const int team_warps = U >= static_cast<long long>(2 * W + kItemUnits) * items ? W : 4;
    const int teams = W / team_warps;
    const int tid = threadIdx.x % (team_warps * 32), wt = warp % team_warps, local = warp / team_warps;
    const int team = local * gridDim.x + blockIdx.x;
    // Heads at a time (all, but where they outnumber the teams), and N groups of that many teams, each with an equal
    // run of units: of a tile a warp or more, since parts cost more to join than idle warps. Heads that wait for a
    // second turn are of one group, which shares no item.
    const int heads = min(a.nkv, static_cast<int>(gridDim.x) * teams);
    const int tiles = U - items * kItemUnits;
    const int N = min((tiles + team_warps - 1) / team_warps, static_cast<int>(gridDim.x) * teams / heads);
    const int group = team / heads;
    if (group >= N) return;
    const int run = U / N, over = U - run * N;
    auto start_of = [&](int k) { return run * k + over * k / N; };
    auto group_of = [&](int u) {  // the last k with start_of(k) <= u
        int lo = 0, hi = N;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start_of(mid) <= u) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    const int u0 = start_of(group), u1 = start_of(group + 1);

    const int G = a.nh / a.nkv;
    int issued = 0, taken = 0;  // tiles of this warp
    bool alive = true;          // false once a bounded wait gave up
    uint8_t* my_ring = ring + warp * kStages * 2 * kTileBytes;
    const uint32_t ring_addr = smem_addr(my_ring), bar_addr = smem_addr(&bars[warp * kStages * 2]);
    for (int kvh = team - group * heads; kvh < a.nkv; kvh += heads) {
    // The fetching end of this warp's tile list: item and tile, the scales of the two tiles in flight, and where the
    // values of a tile whose keys alone are on their way start.
    Item fi = walk.find(u0);
    int fj = max(0, u0 - fi.base) + wt, fend = 0;
    const float *fks = nullptr, *fvs = nullptr;  // scales of the item's first block
    auto enter = [&]() {
        fend = min(fi.tiles, u1 - fi.base);
        const long long at = static_cast<long long>(fi.seq) * a.blocks * a.nkv + kvh;
        fks = a.ks + at;
        fvs = a.vs + at;
    };
    auto settle = [&]() {  // moves on to the item that holds the next tile; false at the end of the run
        while (fj >= fend) {
            if (fi.base + fi.tiles + kItemUnits >= u1) return false;
            walk.next(fi);
            fj = wt;
            enter();
        }
        return true;
    };
    enter();
    const int block_log = 31 - __clz(a.block);
    float ks_q[2][HALVES], vs_q[2][HALVES];  // [0]: the next tile to read, [1]: the one behind it
    int vx = 0, vy = 0;
    bool more = settle();
    auto fetch_keys = [&](float (&ks)[HALVES], float (&vs)[HALVES]) {
        const int st = issued & 1;
        vx = kvh * HD;
        vy = fi.seq * a.max_seq + fj * SLOTS;
        if (lane == 0) {
            bar_expect(bar_addr + 16 * st, kTileBytes);
            tma_load(ring_addr + st * 2 * kTileBytes, &L.kmap, bar_addr + 16 * st, vx, vy);
        }
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int slot = fj * SLOTS + h * 32;
            const long long at = static_cast<long long>(slot >> block_log) * a.nkv;
            const bool holds = slot < fi.len;  // a block behind the sequence has no scale to speak of
            ks[h] = holds ? fks[at] : 0.f;
            vs[h] = holds ? fvs[at] : 0.f;
        }
        ++issued;
        fj += team_warps;
        more = settle();
    };
    auto fetch_values = [&]() {
        if (lane == 0) {
            const int st = (issued - 1) & 1;
            bar_expect(bar_addr + 16 * st + 8, kTileBytes);
            tma_load(ring_addr + st * 2 * kTileBytes + kTileBytes, &L.vmap, bar_addr + 16 * st + 8, vx, vy);
        }
    };
    if (lane == 0) proxy_fence();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!more) break;
        fetch_keys(ks_q[i], vs_q[i]);
        fetch_values();
    }

    Item it = walk.find(u0);
    while (it.base < u1) {  // a run may end before the first tile of its last item
        const int j0 = max(0, u0 - it.base), j1 = min(it.tiles, u1 - it.base);
        const int c0 = it.cg * COLS;  // first column
        const int cols = min(COLS, it.n * G - c0);

        // Query columns: lane (g, t) holds column nt * 8 + g, the dims that its key words will hold, as digits.
        uint32_t qd[NT][KS][ND][2];
        float factor[NT][2];  // score factor of this lane's accumulator columns nt * 8 + 2 t, + 1
        int seen[NT][2];      // slots those columns see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = min(nt * 8 + g, cols - 1);
            float x[HD / 4];
            const int tok = (c0 + col) / G, head = c0 + col - tok * G;
            const T* q = static_cast<const T*>(a.q) + (it.row0 + tok) * a.q_stride + (kvh * G + head) * HD + t * 16;
#pragma unroll
            for (int e = 0; e < HD / 4; e += 8) {
                float y[8];
                load8_f32(q + (e / 16) * 64 + e % 16, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[e + i] = y[i];
            }
            float top = 0.f;
            bool odd = false;  // an infinity or a NaN in the column: its scores become NaN
#pragma unroll
            for (int e = 0; e < HD / 4; ++e) {
                top = fmaxf(top, fabsf(x[e]));
                odd |= !(fabsf(x[e]) < __int_as_float(0x7F800000));
            }
            if (odd) top = __int_as_float(0x7F800000);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^bits lifts the column's largest value to 2^(kTopBit - 1) or more, and at most a top digit of 127.
            int bits = 0;
            if (top > 0.f && top < __int_as_float(0x7F800000)) {
                bits = min(kTopBit - ilogbf(top), 126);
                if (ldexpf(top, bits) > 127.f * (1 << (kTopBit - 6))) --bits;
            }
            float f = ldexpf(a.scale * 1.44269504088896341f, -bits);
            if (top == __int_as_float(0x7F800000)) f = __int_as_float(0x7FC00000);
            const float up = ldexpf(1.f, bits);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    int v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = (__float2int_rn(x[8 * s + 4 * b + i] * up) + kBias) ^ kBias;
#pragma unroll
                    for (int k = 0; k < ND; ++k) qd[nt][s][k][b] = byte_of(v, k);
                }
            }
            factor[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
            factor[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = min(nt * 8 + 2 * t + e, cols - 1);  // columns behind the last repeat it
                seen[nt][e] = max(0, it.len - it.n + (c0 + c) / G + 1);
            }
        }
        const int seen_least = it.len - it.n + c0 / G + 1, seen_most = it.len - it.n + (c0 + cols - 1) / G + 1;

        float o[NT][DT_][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int d = 0; d < DT_; ++d) o[nt][d][0] = o[nt][d][1] = o[nt][d][2] = o[nt][d][3] = 0.f;
            m[nt][0] = m[nt][1] = kNegInf;
            l[nt][0] = l[nt][1] = 0.f;
        }

        bool held = false;  // the stage of this warp's last tile of the segment, kept for the merge
        for (int j = j0 + wt; j < j1; j += team_warps) {
            const int st = taken & 1;
            const uint32_t parity = (taken >> 1) & 1;
            // The last tile's stage stays as it is for the merge; any other's halves are filled again as they are read.
            const bool refill = more && j + team_warps < j1;
            auto wait = [&](uint32_t bar) {
                if (alive && !bar_wait(bar, parity)) {
                    alive = false;
                    if (lane == 0 && a.error) atomicOr(a.error, 1);
                }
                alive = __all_sync(0xffffffffu, alive);
            };
            float ks_n[HALVES], vs_n[HALVES];  // scales of the tile fetched now
#pragma unroll
            for (int h = 0; h < HALVES; ++h) ks_n[h] = vs_n[h] = 0.f;
            wait(bar_addr + 16 * st);
            const int first = j * SLOTS;
            const bool useful = alive && first < seen_most;
            float sc[NT][MT][4];
            // Row r of a score tile is slot row_of(r) of its 16: an order in which the 16-byte reads of keys and of
            // values below both touch every bank once.
            auto row_of = [](int r) { return HD == 128 ? ((r >> 1) | ((r & 1) << 2)) : (r ^ ((r >> 1) & 1)); };
            const uint8_t* kt = my_ring + st * 2 * kTileBytes;
            const uint8_t* vt = kt + kTileBytes;
            if (useful) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    int acc[NT][ND][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < ND; ++k) acc[nt][k][0] = acc[nt][k][1] = acc[nt][k][2] = acc[nt][k][3] = 0;
                    const int ra = mt * 16 + row_of(g);
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) {
                        const int chunk = c * 4 + t;
                        const int phys = HD == 128 ? (chunk ^ (ra & 7)) : (chunk ^ ((ra >> 1) & 3));
                        const uint4 wa = *reinterpret_cast<const uint4*>(kt + ra * HD + phys * 16);
                        const uint4 wb = *reinterpret_cast<const uint4*>(kt + (ra + 8) * HD + phys * 16);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int k = 0; k < ND; ++k) {
                                mma_s8(acc[nt][k], wa.x, wb.x, wa.y, wb.y, qd[nt][2 * c][k][0], qd[nt][2 * c][k][1]);
                                mma_s8(acc[nt][k], wa.z, wb.z, wa.w, wb.w, qd[nt][2 * c + 1][k][0], qd[nt][2 * c + 1][k][1]);
                            }
                        }
                    }
                    // d0 + 256 d1 stays below 2^30, d2 + 256 d3 too: a conversion for each two
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[nt][mt][i] = fmaf(static_cast<float>((ND == 4 ? acc[nt][ND - 1][i] * 256 : 0) + acc[nt][2][i]), 65536.f,
                                                 static_cast<float>(acc[nt][1][i] * 256 + acc[nt][0][i]));
                }
            }
            __syncwarp();  // every lane has read the keys
            if (refill && alive) fetch_keys(ks_n, vs_n);
            if (useful) {
                // Scores in exp2's units, masked; the online softmax of each column.
                float keep[NT][2];
                bool grew = false;
                const bool inside = first + SLOTS <= seen_least;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = kNegInf;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            const float f = factor[nt][e] * ks_q[0][mt / 2];
                            float& x = sc[nt][mt][e];
                            float& y = sc[nt][mt][e + 2];
                            x *= f;
                            y *= f;
                            if (!inside) {
                                const int slot = first + mt * 16 + row_of(g);
                                if (slot >= seen[nt][e]) x = kNegInf;
                                if (slot + 8 >= seen[nt][e]) y = kNegInf;
                            }
                            top = fmaxf(top, fmaxf(x, y));
                        }
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float now = fmaxf(m[nt][e], top);
                        keep[nt][e] = now == m[nt][e] ? 1.f : exp2_fast(m[nt][e] - now);
                        grew |= now != m[nt][e];
                        m[nt][e] = now;
                        const float shift = now == kNegInf ? 0.f : now - kWeightBits;  // nothing seen: weights 0
                        float sum = 0.f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            sc[nt][mt][e] = exp2_fast(sc[nt][mt][e] - shift);
                            sc[nt][mt][e + 2] = exp2_fast(sc[nt][mt][e + 2] - shift);
                            sum += sc[nt][mt][e] + sc[nt][mt][e + 2];
                        }
                        l[nt][e] = fmaf(l[nt][e], keep[nt][e], sum);
                    }
                }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int d = 0; d < DT_; ++d) {
                            o[nt][d][0] *= keep[nt][0];
                            o[nt][d][1] *= keep[nt][1];
                            o[nt][d][2] *= keep[nt][0];
                            o[nt][d][3] *= keep[nt][1];
                        }
                    }
                }
                wait(bar_addr + 16 * st + 8);
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    if (first + h * 32 >= seen_most) break;
                    uint32_t ph[NT][2][2], pl[NT][2][2];  // [k step][b0, b1]
                    float vscale[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float (&s)[4] = sc[nt][2 * h + k];
                            split_f16(s[0], s[1], ph[nt][k][0], pl[nt][k][0]);
                            split_f16(s[2], s[3], ph[nt][k][1], pl[nt][k][1]);
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                ph[nt][k][b] = transposed(ph[nt][k][b]);
                                if constexpr (PAIRS) pl[nt][k][b] = transposed(pl[nt][k][b]);
                            }
                        }
                        // a column that sees none of these slots takes nothing of their scale, whatever it is
#pragma unroll
                        for (int e = 0; e < 2; ++e) vscale[nt][e] = seen[nt][e] > first + h * 32 ? vs_q[0][h] : 0.f;
                    }
                    // Lane (g, t): slots row_of(2 t), row_of(2 t + 1) and those + 8 of each 16, HD / 8 dims from
                    // dim lane_dim on; word w of a slot holds the dims of output tiles 2 w and 2 w + 1.
                    const int lane_dim = HD == 128 ? row_of(g) * 16 : g * 8;
                    uint32_t w[2][4][HD / 32];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = h * 32 + k * 16 + row_of(2 * t + (i & 1)) + (i >> 1) * 8;
                            if constexpr (HD == 128) {
                                const uint4 x = *reinterpret_cast<const uint4*>(vt + r * HD + (((lane_dim >> 4) ^ (r & 7)) << 4));
                                w[k][i][0] = x.x ^ 0x80808080u;
                                w[k][i][1] = x.y ^ 0x80808080u;
                                w[k][i][2] = x.z ^ 0x80808080u;
                                w[k][i][3] = x.w ^ 0x80808080u;
                            } else {
                                const uint2 x = *reinterpret_cast<const uint2*>(
                                    vt + r * HD + (((lane_dim >> 4) ^ ((r >> 1) & 3)) << 4) + (lane_dim & 8));
                                w[k][i][0] = x.x ^ 0x80808080u;
                                w[k][i][1] = x.y ^ 0x80808080u;
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < HD / 32; ++q) {
                        float acc[2][NT][4];
#pragma unroll
                        for (int d = 0; d < 2; ++d)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) acc[d][nt][0] = acc[d][nt][1] = acc[d][nt][2] = acc[d][nt][3] = 0.f;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
#pragma unroll
                            for (int d = 0; d < 2; ++d) {
                                // bytes 2 d, 2 d + 1 of two slots side by side, then each pair as f16
                                const uint32_t x = __byte_perm(w[k][0][q], w[k][1][q], d ? 0x7362 : 0x5140);
                                const uint32_t y = __byte_perm(w[k][2][q], w[k][3][q], d ? 0x7362 : 0x5140);
                                const uint32_t a0 = codes_f16(x, 0x4140), a1 = codes_f16(x, 0x4342);
                                const uint32_t a2 = codes_f16(y, 0x4140), a3 = codes_f16(y, 0x4342);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    mma_f16(acc[d][nt], a0, a1, a2, a3, ph[nt][k][0], ph[nt][k][1]);
                                    if constexpr (PAIRS) mma_f16(acc[d][nt], a0, a1, a2, a3, pl[nt][k][0], pl[nt][k][1]);
                                }
                            }
                        }
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float (&y)[4] = o[nt][2 * q + d];
                                y[0] = fmaf(acc[d][nt][0], vscale[nt][0], y[0]);
                                y[1] = fmaf(acc[d][nt][1], vscale[nt][1], y[1]);
                                y[2] = fmaf(acc[d][nt][2], vscale[nt][0], y[2]);
                                y[3] = fmaf(acc[d][nt][3], vscale[nt][1], y[3]);
                            }
                        }
                    }
                }
            }
            if (!useful) wait(bar_addr + 16 * st + 8);
            ++taken;
            __syncwarp();  // every lane has read the values
            if (refill && alive) fetch_values();
            if (!(j + team_warps < j1)) held = true;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                ks_q[0][h] = ks_q[1][h];
                vs_q[0][h] = vs_q[1][h];
                ks_q[1][h] = ks_n[h];
                vs_q[1][h] = vs_n[h];
            }
        }

        // The segment's end: this warp's state to shared memory, then the team joins the warps' states.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float s = l[nt][e];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                if (g == 0) {
                    ml_s[warp][nt * 8 + 2 * t + e][0] = m[nt][e];
                    ml_s[warp][nt * 8 + 2 * t + e][1] = held ? s : 0.f;
                }
            }
        }
        // Column c, dims 4 x .. 4 x + 3 at 16-byte chunk x ^ ((c >> 1) & 3) of row c: fewer bank conflicts.
        if (held) {
            float* dump = reinterpret_cast<float*>(my_ring + ((taken - 1) & 1) * 2 * kTileBytes);
            const int lane_dim = HD == 128 ? ((g >> 1) | ((g & 1) << 2)) * 16 : g * 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int q = 0; q < HD / 32; ++q) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int c = nt * 8 + 2 * t + e, x = (lane_dim + q * 4) / 4;
                        *reinterpret_cast<float4*>(dump + c * HD + ((x ^ ((c >> 1) & 3)) << 2)) =
                            make_float4(o[nt][2 * q][e], o[nt][2 * q][e + 2], o[nt][2 * q + 1][e], o[nt][2 * q + 1][e + 2]);
                    }
                }
            }
        }
        // Where each warp's dump lies follows from its count of tiles, which the team can work out only for itself:
        // the stage goes with the sums.
        if (lane == 0) last_s[warp] = static_cast<unsigned>((taken - 1) & 1);
        const int bar_id = 1 + local;
        team_sync(bar_id, team_warps * 32);
        const int w0 = local * team_warps;
        const bool whole = j0 == 0 && j1 == it.tiles;
        const int ta = whole ? group : group_of(it.base), tb = whole ? group : group_of(it.base + it.tiles - 1);
        const long long slot = 2LL * team + (group == ta ? 1 : 0);
        for (int e = tid; e < cols * (HD / 4); e += team_warps * 32) {
            const int c = e / (HD / 4), x = e - c * (HD / 4);
            float top = kNegInf;
            for (int w = 0; w < team_warps; ++w) top = fmaxf(top, ml_s[w0 + w][c][0]);
            float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < team_warps; ++w) {
                const float lw = ml_s[w0 + w][c][1];
                if (lw == 0.f) continue;  // nothing seen (a NaN is not 0 and shows)
                const float f = exp2_fast(ml_s[w0 + w][c][0] - top);
                const float* dump = reinterpret_cast<const float*>(ring + ((w0 + w) * kStages + last_s[w0 + w]) * 2 * kTileBytes);
                const float4 y = *reinterpret_cast<const float4*>(dump + c * HD + ((x ^ ((c >> 1) & 3)) << 2));
                sum = fmaf(lw, f, sum);
                v[0] = fmaf(y.x, f, v[0]);
                v[1] = fmaf(y.y, f, v[1]);
                v[2] = fmaf(y.z, f, v[2]);
                v[3] = fmaf(y.w, f, v[3]);
            }
            if (whole) {
                const int tok = (c0 + c) / G, head = c0 + c - tok * G;
                T* out = static_cast<T*>(a.out) + (it.row0 + tok) * a.out_stride + (kvh * G + head) * HD + x * 4;
                // A row without slots gives zeros; one whose every score is -inf has no weights, and 0 / 0 says so.
                const float inv = it.len - it.n + tok < 0 ? 0.f : 1.f / sum;
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(out) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                } else {
                    *reinterpret_cast<uint2*>(out) =
                        make_uint2(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv));
                }
            } else {
                *reinterpret_cast<float4*>(L.part + (slot * COLS + c) * HD + x * 4) = make_float4(v[0], v[1], v[2], v[3]);
                if (x == 0) *reinterpret_cast<float2*>(L.part_ml + (slot * COLS + c) * 2) = make_float2(top, sum);
            }
        }
        if (!whole) {
            team_sync(bar_id, team_warps * 32);
            if (tid == 0) {
                __threadfence();  // after the barrier: for the whole team's writes
                unsigned* arrived = &L.counters[ta * heads + kvh];
                const bool last = atomicAdd(arrived, 1u) == static_cast<unsigned>(tb - ta);
                if (last) *arrived = 0;
                __threadfence();
                last_s[w0] = last ? 2u : 3u;
            }
            team_sync(bar_id, team_warps * 32);
            if (last_s[w0] == 2u) {
                // Parts ta .. tb: the first in its team's last segment, the others in their team's first.
                for (int e = tid; e < cols * (HD / 4); e += team_warps * 32) {
                    const int c = e / (HD / 4), x = e - c * (HD / 4);
                    float top = kNegInf;
                    for (int k = ta; k <= tb; ++k)
                        top = fmaxf(top, __ldcg(L.part_ml + ((2LL * (k * heads + kvh) + (k == ta)) * COLS + c) * 2));
                    float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                    for (int k = ta; k <= tb; ++k) {
                        const long long s = (2LL * (k * heads + kvh) + (k == ta)) * COLS + c;
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(L.part_ml + s * 2));
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(L.part + s * HD + x * 4));
                        const float f = ml.y == 0.f ? 0.f : exp2_fast(ml.x - top);
                        sum = fmaf(ml.y, f, sum);
                        v[0] = fmaf(y.x, f, v[0]);
                        v[1] = fmaf(y.y, f, v[1]);
                        v[2] = fmaf(y.z, f, v[2]);
                        v[3] = fmaf(y.w, f, v[3]);
                    }
                    const int tok = (c0 + c) / G, head = c0 + c - tok * G;
                    T* out = static_cast<T*>(a.out) + (it.row0 + tok) * a.out_stride + (kvh * G + head) * HD + x * 4;
                    const float inv = it.len - it.n + tok < 0 ? 0.f : 1.f / sum;
                    if constexpr (sizeof(T) == 4) {
                        *reinterpret_cast<float4*>(out) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                    } else {
                        *reinterpret_cast<uint2*>(out) =
                            make_uint2(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv));
                    }
                }
            }
        }
        if (it.base + it.tiles + kItemUnits >= u1) break;
        team_sync(bar_id, team_warps * 32);  // the dumps are read: their stages may be filled again
        if (held && more && alive) {
            if (lane == 0) proxy_fence();
            fetch_keys(ks_q[1], vs_q[1]);
            fetch_values();
        }
        walk.next(it);
    }
    team_sync(1 + local, team_warps * 32);
    }
    // A warp that gave up leaves no copy of its own in flight behind it.
    if (!alive) {
        for (; taken < issued; ++taken) {
            bar_wait(bar_addr + 16 * (taken & 1), (taken >> 1) & 1);
            bar_wait(bar_addr + 16 * (taken & 1) + 8, (taken >> 1) & 1);
        }
    }
}

template <typename T, int HD, int NT>
l0b_status launch_q8(l0b_suite* s, l0b_device* d, const AttnQ8Params& a) {
    auto kernel = attn_q8_kernel<T, HD, NT>;
    constexpr int W = warps_of(NT);
    constexpr size_t ring = 1024 + static_cast<size_t>(W) * kStages * 2 * kTileBytes;
    {
        static bool configured[64] = {};
        static std::mutex mu;
        std::lock_guard<std::mutex> lock(mu);
        if (d->index >= 64 || !configured[d->index]) {
            L0B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                static_cast<int>(ring + 4 * (kMaxSequences + 1))));
            if (d->index < 64) configured[d->index] = true;
        }
    }
    // Units are counted in 32 bits: rows of a call times tiles of a cache row, at worst.
    const long long groups = (static_cast<long long>(a.tokens) * (a.nh / a.nkv)) / (8 * NT) + a.count;
    L0B_REQUIRE(groups <= INT32_MAX / (a.max_seq / (kTileBytes / HD) + 1 + kItemUnits), L0B_ERR_OUT_OF_RANGE,
                "%d query rows against %d slots are too many for one call", a.tokens, a.max_seq);
    Q8Launch L;
    std::memset(&L, 0, sizeof L);
    const long long rows = static_cast<long long>(a.count) * a.max_seq, width = static_cast<long long>(a.nkv) * HD;
    const CUtensorMapSwizzle swizzle = HD == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    L0B_TRY(tensor_map_2d(&L.kmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.kc, width, rows, width, HD, kTileBytes / HD, swizzle));
    L0B_TRY(tensor_map_2d(&L.vmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.vc, width, rows, width, HD, kTileBytes / HD, swizzle));
    L.a = a;
    L.part = s->q8_part;
    L.part_ml = s->q8_part + static_cast<size_t>(2 * kQ8TeamsPerSm) * d->sm_count * 16 * 128;
    L.counters = s->q8_counters;
    return d->launch(kernel, dim3(d->sm_count), dim3(W * 32), ring + 4 * (static_cast<size_t>(a.count) + 1), L);
}

template <typename T>
l0b_status launch_as(l0b_suite* s, l0b_device* d, const AttnQ8Params& a) {
    // Two tiles of eight columns where most items fill more than one: each key that is converted then meets both. One tile
    // against two, head dim 128, f16, in us: 16 sequences of up to 4096 slots and 4 KV heads, 9 or 16 columns 35 and 32, 8
    // KV heads of 8 columns 38 and 45; 4 sequences of up to 9001 slots, 14 columns 27 and 29, 35 columns 41 and 41.
    const bool wide = static_cast<long long>(a.nh / a.nkv) * ((a.tokens + a.count - 1) / a.count) > 8;
    if (a.hd == 64) return wide ? launch_q8<T, 64, 2>(s, d, a) : launch_q8<T, 64, 1>(s, d, a);
    return wide ? launch_q8<T, 128, 2>(s, d, a) : launch_q8<T, 128, 1>(s, d, a);
}

}  // namespace

l0b_status k_attention_q8(l0b_suite* s, l0b_device* d, const AttnQ8Params& p) {
    switch (p.dtype) {
        case L0B_F16: return launch_as<__half>(s, d, p);
        case L0B_BF16: return launch_as<__nv_bfloat16>(s, d, p);
        default: return launch_as<float>(s, d, p);
    }
}

}  // namespace l0b
