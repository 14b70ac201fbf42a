// Attention over the int8 KV cache (sm_100a): one CTA per (query row, query head), a thread per key of a tile for
// the scores and a thread per head dimension for the values, online softmax over the tiles.
#include "ops.cuh"
#include "packed.cuh"

namespace l0b {

namespace {

template <typename T, int HD>
__global__ void __launch_bounds__(128) attn_q8_rows_kernel(const AttnQ8Params p) {
    __shared__ float q_s[HD], w_s[128], red[32];
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x, h = blockIdx.y, kvh = h / (p.nh / p.nkv), tid = threadIdx.x;
    const int seq = p.starts ? block_find_sequence(p.starts, p.count, t) : t;
    if (seq < 0) return;
    const int first = p.starts ? p.starts[seq] : seq, end = p.starts ? p.starts[seq + 1] : seq + 1;
    if (t >= end) return;
    const int raw = p.lengths[seq], len = max(0, min(raw, p.max_seq));
    if (tid == 0 && (raw != len || first < 0 || end > p.tokens)) flag_bad_index(p.error);
    const long long seen_raw = static_cast<long long>(len) - end + t + 1;  // keys [0, seen)
    const int seen = static_cast<int>(seen_raw < 0 ? 0 : seen_raw > len ? len : seen_raw);
    const T* q = static_cast<const T*>(p.q) + t * p.q_stride + static_cast<long long>(h) * HD;
    if (tid < HD) q_s[tid] = load_as_float(q, DT<T>::id, tid) * p.scale;
    __syncthreads();
    const int kvd = p.nkv * HD;
    const int8_t* kc = p.kc + static_cast<long long>(seq) * p.max_seq * kvd + kvh * HD;
    const int8_t* vc = p.vc + static_cast<long long>(seq) * p.max_seq * kvd + kvh * HD;
    const float* ks = p.ks + static_cast<long long>(seq) * p.blocks * p.nkv + kvh;
    const float* vs = p.vs + static_cast<long long>(seq) * p.blocks * p.nkv + kvh;
    float m = kNegInf, l = 0.f, acc = 0.f;
    for (int j0 = 0; j0 < seen; j0 += 128) {
        const int j = j0 + tid;
        float s = kNegInf;
        if (j < seen) {
            float dot = 0.f;
            const int8_t* row = kc + static_cast<long long>(j) * kvd;
            for (int d = 0; d < HD; d += 4) {
                float2 a, b;
                dequant_i8x4(*reinterpret_cast<const uint32_t*>(row + d), a, b);
                dot = fmaf(q_s[d], a.x, fmaf(q_s[d + 1], a.y, fmaf(q_s[d + 2], b.x, fmaf(q_s[d + 3], b.y, dot))));
            }
            s = dot * ks[static_cast<long long>(j / p.block) * p.nkv];
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
            for (int i = 0; i < n; ++i)
                acc += w_s[i] * (static_cast<float>(vc[static_cast<long long>(j0 + i) * kvd + tid]) *
                                 vs[static_cast<long long>((j0 + i) / p.block) * p.nkv]);
        }
    }
    if (tid < HD)
        store_from_float(p.out, DT<T>::id, t * p.out_stride + static_cast<long long>(h) * HD + tid, seen > 0 ? acc / l : 0.f);
}

template <typename T>
l0b_status launch_as(l0b_device* d, const AttnQ8Params& p) {
    const dim3 grid(p.tokens, p.nh);
    if (p.hd == 64) return d->launch(attn_q8_rows_kernel<T, 64>, grid, dim3(128), 0, p);
    return d->launch(attn_q8_rows_kernel<T, 128>, grid, dim3(128), 0, p);
}

}  // namespace

l0b_status k_attention_q8(l0b_suite*, l0b_device* d, const AttnQ8Params& p) {
    L0B_REQUIRE(p.nh <= 65535, L0B_ERR_OUT_OF_RANGE, "heads %d exceed 65535", p.nh);
    switch (p.dtype) {
        case L0B_F16: return launch_as<__half>(d, p);
        case L0B_BF16: return launch_as<__nv_bfloat16>(d, p);
        default: return launch_as<float>(d, p);
    }
}

}  // namespace l0b
