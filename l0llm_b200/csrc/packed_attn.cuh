// Shared by the packed-attention kernels (attention_packed.cu, attention_packed_f32.cu): the sequences' extents, the
// scan over them, and the values that a cut tile's guard sets aside.
#pragma once

#include "ops.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace l0b {

l0b_status k_attention_packed_f32(l0b_suite* s, l0b_device* d, const PackedAttnParams& p);

// Rows of one sequence, kept inside the buffers whatever its starts say.
struct PackedSeq {
    int q0, n;  // first query row, query rows
    int k0, m;  // first key row, key rows
};

__device__ __forceinline__ PackedSeq packed_seq(const PackedAttnParams& a, int i) {
    PackedSeq s;
    s.q0 = clamp_start(a.q_starts[i], a.tokens);
    s.n = max(0, clamp_start(a.q_starts[i + 1], a.tokens) - s.q0);
    s.k0 = clamp_start(a.kv_starts[i], a.kv_tokens);
    s.m = max(0, clamp_start(a.kv_starts[i + 1], a.kv_tokens) - s.k0);
    return s;
}

// pre[i] = the sum of units(n) over the sequences before i, pre[count] the total, by the whole CTA. False (and the
// error flag) where the query starts descend: sequences could then share rows of out, which no order of writing settles.
// The answer stays in shared memory (descends_s, 0 before the call): a barrier's own vote would hold a register through the
// f32 path's loop, which then spills (2563 tokens in short prompts: 53.6 -> 61 us).
template <typename F>
__device__ __forceinline__ bool packed_scan(const PackedAttnParams& a, int* pre, int* warp_sums, int* descends_s, F units) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int per = (a.count + blockDim.x - 1) / blockDim.x, i0 = threadIdx.x * per, i1 = min(a.count, i0 + per);
    int mine = 0;
    bool bad = false, descends = false;
    for (int i = i0; i < i1; ++i) {
        mine += units(packed_seq(a, i).n);
        descends |= a.q_starts[i] > a.q_starts[i + 1];
        bad |= descends || a.q_starts[i] < 0 || a.q_starts[i + 1] > a.tokens || a.kv_starts[i] < 0 ||
               a.kv_starts[i + 1] > a.kv_tokens || a.kv_starts[i] > a.kv_starts[i + 1];
    }
    if (bad && blockIdx.x == 0) flag_bad_index(a.error);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sums[warp] = sum;
    if (descends) atomicOr(descends_s, 1);
    __syncthreads();
    const bool fine = *descends_s == 0;
    int before = sum - mine;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    for (int i = i0; i < i1; ++i) {
        pre[i] = before;
        before += units(packed_seq(a, i).n);
    }
    if (threadIdx.x == 0) {
        int all = 0;
        for (int w = 0; w < warps; ++w) all += warp_sums[w];
        pre[a.count] = all;
    }
    __syncthreads();
    return fine;
}

// Whether one of eight 16-bit values is an infinity or a NaN: an exponent of ones carries into the bit above it.
template <bool BF>
__device__ __forceinline__ bool not_finite(const uint4& w) {
    const uint32_t mask = BF ? 0x7F807F80u : 0x7C007C00u, one = BF ? 0x00800080u : 0x04000400u;
    return ((((w.x & mask) + one) | ((w.y & mask) + one) | ((w.z & mask) + one) | ((w.w & mask) + one)) & 0x80008000u) != 0;
}

// Makes 64 value rows of a cut tile, base on, safe for weights of 0, by one warp: rows from `live` on (another sequence's)
// and rows with an infinity or a NaN become zeros; the latter are noted in bad. v: BLOCKS swizzled blocks of 64 columns.
template <bool BF, int BLOCKS>
__device__ __forceinline__ void guard_rows(uint8_t* v, int base, int live, int lane, uint32_t (&bad)[2]) {
    // A row takes LANES lanes of 16 bytes; the warp looks at AT_ONCE rows a step, eight steps in flight.
    constexpr int LANES = BLOCKS * 8, AT_ONCE = 32 / LANES;
    const int sub = lane / LANES, c = lane % LANES;
    bad[0] = bad[1] = 0;
#pragma unroll 1
    for (int r0 = 0; r0 < 64; r0 += 8 * AT_ONCE) {
        uint8_t* at = v + (c >> 3) * kSub + (base + r0 + sub) * 128 + (c & 7) * 16;
        uint32_t odd = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint4 w = *reinterpret_cast<const uint4*>(at + k * AT_ONCE * 128);
            odd |= static_cast<uint32_t>(not_finite<BF>(w) && base + r0 + k * AT_ONCE + sub < live) << k;
        }
        if (!__any_sync(0xffffffffu, odd != 0) && base + r0 + 8 * AT_ONCE <= live) continue;
        for (int k = 0; k < 8; ++k) {
            const uint32_t hit = __ballot_sync(0xffffffffu, (odd >> k) & 1);
            const uint32_t row_mask = (1u << LANES) - 1u;
            if (((hit >> (sub * LANES)) & row_mask) || base + r0 + k * AT_ONCE + sub >= live)
                *reinterpret_cast<uint4*>(at + k * AT_ONCE * 128) = make_uint4(0, 0, 0, 0);
            for (int q = 0; q < AT_ONCE; ++q) {
                const int r = r0 + k * AT_ONCE + q;
                if ((hit >> (q * LANES)) & row_mask) bad[r >> 5] |= 1u << (r & 31);
            }
        }
    }
}

// The weight exp2((q . k) c - shift) of one key for one query row, worked out anew: for the few values that are not
// finite in tiles that the mask cuts.
template <typename T, int HD>
__device__ __noinline__ float weight_anew(const PackedAttnParams& a, const PackedSeq& s, int head, int row, int key, float c,
                                          float shift) {
    const T* k = static_cast<const T*>(a.k) + static_cast<long long>(s.k0 + key) * a.k_stride + head / (a.nh / a.nkv) * HD;
    const long long q = static_cast<long long>(s.q0 + row) * a.q_stride + static_cast<long long>(head) * HD;
    float dot = 0.f;
    for (int d = 0; d < HD; ++d) dot = fmaf(load_as_float(a.q, a.q_dtype, q + d), load_as_float(k, DT<T>::id, d), dot);
    return exp2f(dot * c - shift);
}

}  // namespace l0b
