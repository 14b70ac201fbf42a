// The int8 KV cache with one scale per (block of slots, KV head): store and load (sm_100a).
//
// Store. One CTA owns the block pieces that start in its range of packed rows (a piece: the rows of one
// sequence that land in one block of slots; the row that opens it is its leader), for one KV head of K or V.
// Every new value of a piece stays in registers between the two things done with it: the largest magnitude
// (bits of |x| compared as integers, so an infinity or a NaN wins and the scale shows it) and the codes. So
// the rows are read once and the codes written once; both are bound by HBM.
//
// scale = f32(max / 127), never below the old one where slots of the block below the piece are kept.
// code = rint(x / scale) of the exact quotient: q = rint(x * (1 / scale)) may be one off next to a half, and
// the residual x - q * scale decides. In f32 fma that residual is exact wherever it is near scale / 2 (x and
// q * scale are multiples of ulp(scale) there, or x is below scale and within a factor of two of it), so
// 2 |r| compares with scale as the real numbers do; a tie goes to the even code.
#include "ops.cuh"
#include "packed.cuh"

namespace l0b {

namespace {

constexpr int kPer = 32;  // values of a piece per thread: threads = block * hd / 32

__device__ __forceinline__ int code_of(float x, float scale, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, scale, x), twice = 2.f * fabsf(r);
    const float toward = r < 0.f ? -1.f : 1.f;
    if (twice > scale || (twice == scale && (static_cast<int>(q) & 1))) q += toward;
    return static_cast<int>(fminf(127.f, fmaxf(-127.f, q)));
}

// The same by f64, where 1 / scale has no f32 or x is an old code times its old scale: a quotient of at most
// 2^31 / 2^24 that is not a half is further from it than f64's rounding.
__device__ __forceinline__ int code_of_f64(double x, float scale) {
    return static_cast<int>(fmin(127.0, fmax(-127.0, rint(x / static_cast<double>(scale)))));
}

template <typename T, int HD>
__global__ void __launch_bounds__(512) kv_q8_store_kernel(const KvQ8Params p, int rows_per_cta) {
    __shared__ unsigned red[32];
    const int head = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int kvd = p.nkv * HD;
    const T* src = static_cast<const T*>(which ? p.v : p.k) + head * HD;
    const long long stride = which ? p.v_stride : p.k_stride;
    int8_t* cache = (which ? p.vc : p.kc) + head * HD;
    float* scales = (which ? p.vs : p.ks) + head;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    pdl_wait();
    pdl_launch_dependents();

    const int t0 = blockIdx.x * rows_per_cta, t1 = min(p.tokens, t0 + rows_per_cta);
    int seq = p.starts ? block_find_sequence(p.starts, p.count, t0) : t0;
    if (seq < 0) seq = 0;  // rows before the first sequence; a sequence may still start inside the range
    for (; seq < p.count; ++seq) {
        const int first = p.starts ? p.starts[seq] : seq, end_raw = p.starts ? p.starts[seq + 1] : seq + 1;
        if (first >= t1) break;
        const int pos = p.positions[seq];
        const int end = min(end_raw, p.tokens);
        if (first < 0 || end_raw > p.tokens || pos < 0 || (end > first && pos > p.max_seq - (end - first))) {
            if (tid == 0) flag_bad_index(p.error);
            if (first < 0 || pos < 0 || pos >= p.max_seq) continue;
        }
        const int stop = min(end - first, p.max_seq - pos) + pos;  // past the sequence's last new slot
        // Leaders of this sequence in [t0, t1): its first row, then every row that opens a block.
        long long t = first;
        if (t < t0) t = t0 + (p.block - (pos + static_cast<long long>(t0 - first)) % p.block) % p.block;
        while (t < min(end, t1) && pos + (t - first) < stop) {
            const int slot = static_cast<int>(pos + (t - first));
            const int blk = slot / p.block, base = blk * p.block;
            const int last = min(base + p.block, stop);  // past the piece's last new slot
            const int n = last - slot;
            // Values of the piece: thread holds four groups of eight, group g at element (g * threads + tid) * 8.
            float x[4][8];
            unsigned top = 0;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int e = (g * blockDim.x + tid) * 8, r = e / HD, c = e % HD;
                if (r < n) {
                    load8_f32(src + (t + r) * stride + c, x[g]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[g][i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[g][i]) & 0x7FFFFFFFu);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            __syncthreads();
            if (lane == 0) red[warp] = top;
            __syncthreads();
            top = __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
            float* sp = scales + (static_cast<long long>(seq) * p.blocks + blk) * p.nkv;
            float scale = __fdiv_rn(__uint_as_float(top), 127.f), old = 0.f;
            const int kept = slot - base;
            if (kept > 0) {
                old = *sp;
                const unsigned ob = __float_as_uint(old) & 0x7FFFFFFFu, nb = __float_as_uint(scale);
                scale = __uint_as_float(max(ob, nb));
            }
            const bool fine = scale > 0.f && scale < __int_as_float(0x7F800000);
            int8_t* dst = cache + (static_cast<long long>(seq) * p.max_seq + base) * kvd;
            if (kept > 0 && __float_as_uint(scale) != __float_as_uint(old)) {
                for (int e = tid * 8; e < kept * HD; e += blockDim.x * 8) {
                    const int r = e / HD, c = e % HD;
                    uint2* at = reinterpret_cast<uint2*>(dst + static_cast<long long>(r) * kvd + c);
                    const uint2 was = *at;
                    uint32_t w[2] = {was.x, was.y};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t u = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c8 = static_cast<int8_t>(w[k] >> (8 * i));
                            const int q = fine ? code_of_f64(c8 * static_cast<double>(old), scale) : 0;
                            u |= (static_cast<uint32_t>(q) & 0xFFu) << (8 * i);
                        }
                        w[k] = u;
                    }
                    *at = make_uint2(w[0], w[1]);
                }
            }
            const float inv = 1.f / scale;
            const bool quick = fine && scale > 1e-36f;  // 1 / scale and twice the residual are normal numbers
            dst += static_cast<long long>(kept) * kvd;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int e = (g * blockDim.x + tid) * 8, r = e / HD, c = e % HD;
                if (r >= n) continue;
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int q = quick ? code_of(x[g][i], scale, inv) : fine ? code_of_f64(x[g][i], scale) : 0;
                    w[i >> 2] |= (static_cast<uint32_t>(q) & 0xFFu) << (8 * (i & 3));
                }
                *reinterpret_cast<uint2*>(dst + static_cast<long long>(r) * kvd + c) = make_uint2(w[0], w[1]);
            }
            __syncthreads();  // every thread has read the old scale
            if (tid == 0) *sp = scale;
            t += n;
        }
    }
}

// Load. A CTA takes `rows` packed rows; each thread turns sixteen codes at a time into values. Bound by HBM.
template <typename T>
__global__ void __launch_bounds__(256) kv_q8_load_kernel(const KvQ8Params p, int rows) {
    __shared__ int slot_of[32], seq_of[32];
    pdl_wait();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * rows, n = min(rows, p.tokens - t0);
    const int s0 = p.starts ? block_find_sequence(p.starts, p.count, t0) : t0;
    if (threadIdx.x < n) {
        const int t = t0 + threadIdx.x;
        int seq = p.starts ? max(s0, 0) : t, slot = -1;
        if (p.starts) {
            while (seq + 1 < p.count && p.starts[seq + 1] <= t) ++seq;
        }
        const int first = p.starts ? p.starts[seq] : seq, end = p.starts ? p.starts[seq + 1] : seq + 1;
        if (t >= first && t < end) {
            const int pos = p.positions[seq];
            if (pos < 0 || first < 0 || end > p.tokens || pos >= p.max_seq - (t - first)) flag_bad_index(p.error);
            if (pos >= 0 && pos < p.max_seq - (t - first)) slot = pos + (t - first);
        }
        slot_of[threadIdx.x] = slot;
        seq_of[threadIdx.x] = seq;
    }
    __syncthreads();
    const int kvd = p.nkv * p.hd, per_row = kvd / 16;
    for (int e = threadIdx.x; e < n * per_row * 2; e += 256) {
        const int which = e >= n * per_row;
        const int i = which ? e - n * per_row : e;
        const int r = i / per_row, c = (i - r * per_row) * 16;
        const int slot = slot_of[r], seq = seq_of[r];
        if (slot < 0) continue;
        const int8_t* src = (which ? p.vc : p.kc) + (static_cast<long long>(seq) * p.max_seq + slot) * kvd + c;
        const float scale = (which ? p.vs : p.ks)[(static_cast<long long>(seq) * p.blocks + slot / p.block) * p.nkv + c / p.hd];
        const uint4 w4 = ld_stream_v4(src);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        T* dst = static_cast<T*>(const_cast<void*>(which ? p.v : p.k)) + (t0 + r) * (which ? p.v_stride : p.k_stride) + c;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float2 a, b;
                dequant_i8x4(w[2 * h + j], a, b);
                v[4 * j] = a.x * scale;
                v[4 * j + 1] = a.y * scale;
                v[4 * j + 2] = b.x * scale;
                v[4 * j + 3] = b.y * scale;
            }
            store8(dst + 8 * h, v);
        }
    }
}

template <typename T>
l0b_status store_as(l0b_device* d, const KvQ8Params& p) {
    const int threads = p.block * p.hd / kPer;  // 64 .. 512
    // Packed rows per CTA: a block's worth where that alone fills the SMs (the leaders of a range run in
    // turn), fewer for short runs, one for a decode step.
    const long long pieces = static_cast<long long>(p.tokens) * p.nkv * 2;
    int rows = p.starts ? p.block : 1;
    while (rows > 1 && pieces / rows < 8LL * d->sm_count) rows >>= 1;
    const dim3 grid((p.tokens + rows - 1) / rows, p.nkv * 2);
    L0B_REQUIRE(p.nkv <= 32767, L0B_ERR_OUT_OF_RANGE, "KV heads %d exceed 32767", p.nkv);
    if (p.hd == 64) return d->launch(kv_q8_store_kernel<T, 64>, grid, dim3(threads), 0, p, rows);
    return d->launch(kv_q8_store_kernel<T, 128>, grid, dim3(threads), 0, p, rows);
}

template <typename T>
l0b_status load_as(l0b_device* d, const KvQ8Params& p) {
    int rows = 32;
    while (rows > 1 && p.tokens / rows < 4 * d->sm_count) rows >>= 1;
    return d->launch(kv_q8_load_kernel<T>, dim3((p.tokens + rows - 1) / rows), dim3(256), 0, p, rows);
}

}  // namespace

l0b_status k_kv_q8_store(l0b_device* d, const KvQ8Params& p) {
    switch (p.dtype) {
        case L0B_F16: return store_as<__half>(d, p);
        case L0B_BF16: return store_as<__nv_bfloat16>(d, p);
        default: return store_as<float>(d, p);
    }
}

l0b_status k_kv_q8_load(l0b_device* d, const KvQ8Params& p) {
    switch (p.dtype) {
        case L0B_F16: return load_as<__half>(d, p);
        case L0B_BF16: return load_as<__nv_bfloat16>(d, p);
        default: return load_as<float>(d, p);
    }
}

}  // namespace l0b
