// Causal attention over packed sequences, f32 queries (sm_100a): one CTA per (query row, query head), a thread per key of a tile
// for the scores and a thread per head dimension for the values, online softmax over the tiles.
#include "ops.cuh"
#include "packed.cuh"
#include "packed_attn.cuh"

namespace l0b {

namespace {

template <typename TQ, typename TK, int HD>
__global__ void __launch_bounds__(128) attn_packed_rows_kernel(const PackedAttnParams p) {
    __shared__ float q_s[HD], w_s[128], red[32];
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x, h = blockIdx.y, kvh = h / (p.nh / p.nkv), tid = threadIdx.x;
    const int seq = block_find_sequence(p.q_starts, p.count, t);
    if (seq < 0) return;
    const int first = p.q_starts[seq], end = p.q_starts[seq + 1];
    if (t >= end) return;
    const int k0_raw = p.kv_starts[seq], k1_raw = p.kv_starts[seq + 1];
    const int k0 = max(0, min(k0_raw, p.kv_tokens)), m_keys = max(0, min(k1_raw, p.kv_tokens) - k0);
    if (tid == 0 && (first < 0 || end > p.tokens || k0_raw != k0 || k1_raw != k0 + m_keys)) flag_bad_index(p.error);
    const long long seen_raw = static_cast<long long>(m_keys) - end + t + 1;
    const int seen = static_cast<int>(seen_raw < 0 ? 0 : seen_raw > m_keys ? m_keys : seen_raw);
    const TQ* q = static_cast<const TQ*>(p.q) + t * p.q_stride + static_cast<long long>(h) * HD;
    if (tid < HD) q_s[tid] = load_as_float(q, DT<TQ>::id, tid) * p.scale;
    __syncthreads();
    const TK* k = static_cast<const TK*>(p.k) + k0 * p.k_stride + kvh * HD;
    const TK* v = static_cast<const TK*>(p.v) + k0 * p.v_stride + kvh * HD;
    float m = kNegInf, l = 0.f, acc = 0.f;
    for (int j0 = 0; j0 < seen; j0 += 128) {
        const int j = j0 + tid;
        float s = kNegInf;
        if (j < seen) {
            s = 0.f;
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                load8_f32(k + j * p.k_stride + d, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(q_s[d + i], x[i], s);
            }
        }
        float top = warp_max(s);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float next = fmaxf(m, top), keep = m == kNegInf ? 0.f : expf(m - next);
        const float w = j < seen ? expf(s - next) : 0.f;
        m = next;
        l = l * keep + block_sum(w, red);
        w_s[tid] = w;
        __syncthreads();
        acc *= keep;
        if (tid < HD) {
            const int n = min(128, seen - j0);
            for (int i = 0; i < n; ++i) acc += w_s[i] * load_as_float(v + (j0 + i) * p.v_stride, DT<TK>::id, tid);
        }
    }
    if (tid < HD)
        store_from_float(p.out, DT<TQ>::id, t * p.out_stride + static_cast<long long>(h) * HD + tid, seen > 0 ? acc / l : 0.f);
}

template <typename TQ, typename TK>
l0b_status launch_as(l0b_device* d, const PackedAttnParams& p) {
    const dim3 grid(p.tokens, p.nh);
    if (p.hd == 64) return d->launch(attn_packed_rows_kernel<TQ, TK, 64>, grid, dim3(128), 0, p);
    return d->launch(attn_packed_rows_kernel<TQ, TK, 128>, grid, dim3(128), 0, p);
}

}  // namespace

l0b_status k_attention_packed_f32(l0b_suite*, l0b_device* d, const PackedAttnParams& p) {
    L0B_REQUIRE(p.nh <= 65535, L0B_ERR_OUT_OF_RANGE, "heads %d exceed 65535", p.nh);
    return p.kv_dtype == L0B_F16 ? launch_as<float, __half>(d, p) : launch_as<float, __nv_bfloat16>(d, p);
}

}  // namespace l0b
