// The int8 KV cache with one scale per (block of slots, KV head): store and load (sm_100a).
//
// Store. One CTA owns the block pieces that start in its range of packed rows (a piece: the rows of one
// sequence that land in one block of slots; the row that opens it is its leader), for one KV head of K or V.
// Every new value of a piece stays in registers between the two things done with it: the largest magnitude
// (bits of |x| compared as integers, so an infinity or a NaN wins and the scale shows it) and the codes. So
// the rows are read once and the codes written once. 22,167 bf16 rows of 8 heads of 128 take 35 us, 3.9 TB/s: a piece
// is a chain of a fetch, a maximum over the CTA and a write, and two CTAs an SM (64 registers) hide some of it; three of
// 40 registers spill and took 7% longer.
//
// scale = f32(max / 127), never below the old one where slots of the block below the piece are kept.
// code = rint(x / scale) of the exact quotient: the nearest integer q to x * (1 / scale) may be one off next to a half,
// and the residual x - q * scale decides. In f32 fma that residual is exact wherever it is near scale / 2 (x and
// q * scale are multiples of ulp(scale) there, or x is below scale and within a factor of two of it), so |r| compares
// with scale / 2 as the real numbers do; a tie goes to the even code.
#include "ops.cuh"
#include "packed.cuh"

namespace l0b {

namespace {

constexpr int kPer = 32;  // values of a piece per thread: threads = block * hd / 32

// rint(x / scale) of the exact quotient by f64, for scales whose reciprocal is no normal f32 and for x an old code
// times its old scale: a quotient of numbers of 31 and 24 bits that is not a half is further from one than f64 rounds.
__device__ __forceinline__ int code_of_f64(double x, float scale) {
    return static_cast<int>(fmin(127.0, fmax(-127.0, rint(x / static_cast<double>(scale)))));
}

// Starts outside the rows or descending may leave rows to nobody, who then could not report it. The last CTA looks at
// all starts and does nothing else: in one that also works the first and the last alone cost 2 us of cold loads.
__device__ __forceinline__ void check_starts(const KvQ8Params& p) {
    if (!p.starts) return;
    bool bad = false;
    for (int i = threadIdx.x; i <= p.count; i += blockDim.x) {
        const int start = p.starts[i], next = p.starts[min(i + 1, p.count)];
        bad |= start != clamp_start(start, p.tokens) || start > next;
    }
    if (bad) flag_bad_index(p.error);
}

template <typename T>
__device__ __forceinline__ float2 pair_of(const uint32_t* w, int i) {  // values 2 i, 2 i + 1
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return DT<T>::id == L0B_F16 ? half2_bits_to_float2(w[i]) : bf162_bits_to_float2(w[i]);
}

// Codes of the slots [0, kept) of a block from one scale to another.
__device__ __noinline__ void rescale_kept(int8_t* block, int kvd, int hd_log, int kept, float old, float scale, bool fine) {
    for (int e = threadIdx.x * 8; e < kept << hd_log; e += blockDim.x * 8) {
        uint2* at = reinterpret_cast<uint2*>(block + static_cast<long long>(e >> hd_log) * kvd + (e & ((1 << hd_log) - 1)));
        const uint2 was = *at;
        uint32_t w[2] = {was.x, was.y};
        for (int k = 0; k < 2; ++k) {
            uint32_t u = 0;
            for (int i = 0; i < 32; i += 8) {
                const int c = static_cast<int8_t>(w[k] >> i);
                u |= (static_cast<uint32_t>(fine ? code_of_f64(c * static_cast<double>(old), scale) : 0) & 0xFFu) << i;
            }
            w[k] = u;
        }
        *at = make_uint2(w[0], w[1]);
    }
}

// Codes of a piece of n rows by f64, or 0 where the scale is 0 or not finite; the rows are read again.
template <typename T, int HD>
__device__ __noinline__ void store_slowly(const T* src, long long stride, int8_t* dst, int kvd, int n, float scale, bool fine) {
    for (int e = threadIdx.x; e < n * HD; e += blockDim.x) {
        const int r = e / HD, c = e % HD;
        dst[static_cast<long long>(r) * kvd + c] =
            static_cast<int8_t>(fine ? code_of_f64(load_as_float(src, DT<T>::id, r * stride + c), scale) : 0);
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(512, 2) kv_q8_store_kernel(const KvQ8Params p, int rows_per_cta) {
    constexpr int WORDS = 8 * sizeof(T) / 4;  // of eight values
    __shared__ unsigned red[32];
    // The heads of the same rows side by side: together they read and write whole rows while their DRAM pages are open.
    const int range = blockIdx.x / (2 * p.nkv), hw = blockIdx.x - range * 2 * p.nkv, head = hw >> 1, which = hw & 1;
    const int kvd = p.nkv * HD;
    const T* src = static_cast<const T*>(which ? p.v : p.k) + head * HD;
    const long long stride = which ? p.v_stride : p.k_stride;
    int8_t* cache = (which ? p.vc : p.kc) + head * HD;
    float* scales = (which ? p.vs : p.ks) + head;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
    const int block_log = 31 - __clz(p.block);
    const int row0 = tid / (HD / 8), col = tid % (HD / 8) * 8, step = blockDim.x / (HD / 8);
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x == gridDim.x - 1) return check_starts(p);

    const int t0 = range * rows_per_cta, t1 = min(p.tokens, t0 + rows_per_cta);
    int seq = p.starts ? block_find_sequence(p.starts, p.count, t0) : t0;
    if (seq < 0) seq = 0;  // rows before the first sequence; a sequence may still start inside the range
    for (; seq < p.count; ++seq) {
        const int first = p.starts ? p.starts[seq] : seq, end_raw = p.starts ? p.starts[seq + 1] : seq + 1;
        if (first >= t1) break;
        const int pos = p.positions[seq];
        const int end = clamp_start(end_raw, p.tokens);
        if (first < 0 || end_raw > p.tokens || pos < 0 || (end > first && pos > p.max_seq - (end - first))) {
            if (tid == 0) flag_bad_index(p.error);
            if (first < 0 || pos < 0 || pos >= p.max_seq) continue;
        }
        const int stop = min(end - first, p.max_seq - pos) + pos;  // past the sequence's last new slot
        // Leaders of this sequence in [t0, t1): its first row, then every row that opens a block.
        long long t = first;
        if (t < t0) t = t0 + static_cast<int>(-(static_cast<unsigned>(pos) + (t0 - first)) & (p.block - 1));
        while (t < min(end, t1) && pos + (t - first) < stop) {
            const int slot = static_cast<int>(pos + (t - first));
            const int blk = slot >> block_log, base = blk << block_log;
            const int n = min(base + p.block, stop) - slot, kept = slot - base;
            // Values of the piece: a thread holds eight columns from `col` on of four rows, `step` apart.
            const T* from = src + (t + row0) * stride + col;
            uint32_t w[4][WORDS];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int i = 0; i < WORDS; i += 4) {
                    uint4 u = make_uint4(0, 0, 0, 0);
                    if (row0 + g * step < n) u = ld_once_v4(from + i * 4 / static_cast<int>(sizeof(T)));
                    w[g][i] = u.x;
                    w[g][i + 1] = u.y;
                    w[g][i + 2] = u.z;
                    w[g][i + 3] = u.w;
                }
                from += step * stride;
            }
            float* sp = scales + (static_cast<long long>(seq) * p.blocks + blk) * p.nkv;
            const float old = kept > 0 ? *sp : 0.f;
            unsigned top = 0;  // the largest magnitude's bits: an infinity is above every number, a NaN above that
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
                for (int i = 0; i < WORDS; i += 2) {
                    if constexpr (sizeof(T) == 4) top = __vimax3_u32(top, w[g][i] & 0x7FFFFFFFu, w[g][i + 1] & 0x7FFFFFFFu);
                    else top = __vimax3_u16x2(top, w[g][i] & 0x7FFF7FFFu, w[g][i + 1] & 0x7FFF7FFFu);
                }
            }
            if constexpr (sizeof(T) == 2) {  // the larger half, as f32 bits
                const float2 both = pair_of<T>(&top, 0);
                top = max(__float_as_uint(both.x), __float_as_uint(both.y));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            __syncthreads();
            if (lane == 0) red[warp] = top;
            __syncthreads();  // and every thread has read the old scale
            top = __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
            float scale = __fdiv_rn(__uint_as_float(top), 127.f);
            if (kept > 0) scale = __uint_as_float(max(__float_as_uint(old) & 0x7FFFFFFFu, __float_as_uint(scale)));
            const bool fine = scale > 0.f && scale < __int_as_float(0x7F800000);
            int8_t* dst = cache + (static_cast<long long>(seq) * p.max_seq + base) * kvd;
            dst += static_cast<long long>(kept) * kvd;
            if (fine && scale > 1e-36f) {  // the reciprocal and every residual next to a half are normal numbers
                const float half = 0.5f * scale, inv1 = 1.f / scale;
                const float2 inv = make_float2(inv1, inv1), minus = make_float2(-scale, -scale);
                const float2 magic = make_float2(12582912.f, 12582912.f), unmagic = make_float2(-12582912.f, -12582912.f);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t q[8];
                    float worst = 0.f, res[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // 1.5 2^23 + the nearest integer: its low byte is the code
                        const float2 x = pair_of<T>(w[g], i);
                        const float2 n = ffma2(x, inv, magic), r = ffma2(fadd2(n, unmagic), minus, x);
                        res[2 * i] = r.x;
                        res[2 * i + 1] = r.y;
                        q[2 * i] = __float_as_uint(n.x);
                        q[2 * i + 1] = __float_as_uint(n.y);
                        worst = fmaxf(fmaxf(worst, fabsf(res[2 * i])), fabsf(res[2 * i + 1]));
                    }
                    // next to a half, which is rare: a branch of the warp
                    if (__any_sync(0xffffffffu, worst >= half)) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float d = fabsf(res[i]);
                            if (d > half || (d == half && (q[i] & 1))) q[i] += res[i] < 0.f ? -1 : 1;
                        }
                    }
                    uint2 out;
                    out.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                    out.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
                    if (row0 + g * step < n)
                        *reinterpret_cast<uint2*>(dst + static_cast<long long>(row0 + g * step) * kvd + col) = out;
                }
            } else {
                store_slowly<T, HD>(src + t * stride, stride, dst, kvd, n, scale, fine);
            }
            if (kept > 0 && __float_as_uint(scale) != __float_as_uint(old))  // last: nothing else is held over the call
                rescale_kept(dst - static_cast<long long>(kept) * kvd, kvd, HD == 128 ? 7 : 6, kept, old, scale, fine);
            if (tid == 0) *sp = scale;
            t += n;
        }
    }
}

// Load. A warp takes one packed row, K and V of it: 128 or 256 codes a step into 512 contiguous bytes. Bound by HBM:
// 76,545 rows of 8 heads of 128 as f16 take 73 us, 6.4 TB/s; 86 before four steps' codes were loaded ahead of the first
// step's stores. (Warps that took a run of rows, to find their sequence once, were no faster, and slower for 4000 short
// sequences, 194 against 156 us; finding one of 4096 takes three reads.)
template <typename T>
__global__ void __launch_bounds__(256) kv_q8_load_kernel(const KvQ8Params p) {
    constexpr int VEC = 16 / sizeof(T);  // codes of a thread's step: 16 bytes out
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x == gridDim.x - 1) return check_starts(p);
    const int lane = threadIdx.x & 31, t = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int kvd = p.nkv * p.hd, hd_log = p.hd == 128 ? 7 : 6, block_log = 31 - __clz(p.block);
    if (t >= p.tokens) return;
    int seq = t, first = t;
    if (p.starts) {  // the last sequence that starts at or before the row: each step looks at 32 of those left
        int before = 0, left = p.count;
        while (left > 0) {
            const int step = (left + 31) / 32, i = before + (lane + 1) * step - 1;
            const int n = step * __popc(__ballot_sync(0xffffffffu, i < before + left && p.starts[i] <= t));
            before += n;
            left = min(left - n, step - 1);
        }
        seq = before - 1;
        if (seq < 0) return;
        first = p.starts[seq];
        const int end = p.starts[seq + 1];
        if (lane == 0 && (first < 0 || end > p.tokens)) flag_bad_index(p.error);
        if (t >= end) return;
    }
    const int pos = p.positions[seq];
    const long long nth = static_cast<long long>(t) - first;  // a start may be any number
    if (pos < 0 || nth < 0 || pos + nth >= p.max_seq) {       // in front of its sequence: starts that descend
        if (lane == 0) flag_bad_index(p.error);
        return;
    }
    const int slot = pos + static_cast<int>(nth);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int8_t* src = (which ? p.vc : p.kc) + (static_cast<long long>(seq) * p.max_seq + slot) * kvd;
        const float* scales = (which ? p.vs : p.ks) + (static_cast<long long>(seq) * p.blocks + (slot >> block_log)) * p.nkv;
        T* dst = static_cast<T*>(const_cast<void*>(which ? p.v : p.k)) + t * (which ? p.v_stride : p.k_stride);
        // Four steps' codes and scales are on their way before the first is written.
        for (int c0 = lane * VEC; c0 < kvd; c0 += 4 * 32 * VEC) {
            uint32_t w[4][VEC / 4];
            float scale[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = c0 + k * 32 * VEC;
                if (c >= kvd) break;
                if constexpr (VEC == 4) {
                    w[k][0] = *reinterpret_cast<const unsigned*>(src + c);
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(src + c);
                    w[k][0] = u.x;
                    w[k][1] = u.y;
                }
                scale[k] = scales[c >> hd_log];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = c0 + k * 32 * VEC;
                if (c >= kvd) break;
                float v[8];
#pragma unroll
                for (int j = 0; j < VEC / 4; ++j) {
                    float2 a, b;
                    dequant_i8x4(w[k][j], a, b);
                    v[4 * j] = a.x * scale[k];
                    v[4 * j + 1] = a.y * scale[k];
                    v[4 * j + 2] = b.x * scale[k];
                    v[4 * j + 3] = b.y * scale[k];
                }
                // f32 rows go past the L2: 22,167 rows stored and read back 78.5 -> 70.7 us. 16-bit ones would lose 1%.
                if constexpr (VEC == 4) __stcs(reinterpret_cast<float4*>(dst + c), make_float4(v[0], v[1], v[2], v[3]));
                else store8(dst + c, v);
            }
        }
    }
}

template <typename T>
l0b_status store_as(l0b_device* d, const KvQ8Params& p) {
    const int threads = p.block * p.hd / kPer;  // 64 .. 512
    // Packed rows per CTA: two blocks' worth where that alone fills the SMs (the leaders of a range run in turn; one
    // block a CTA took 3% longer, four and eight 2% and 8%), fewer for short runs, one for a decode step.
    const long long pieces = static_cast<long long>(p.tokens) * p.nkv * 2;
    int rows = p.starts ? 2 * p.block : 1;
    while (rows > 1 && pieces / rows < 8LL * d->sm_count) rows >>= 1;
    const long long ctas = (static_cast<long long>(p.tokens) + rows - 1) / rows * p.nkv * 2;
    L0B_REQUIRE(ctas < INT32_MAX, L0B_ERR_OUT_OF_RANGE, "%d rows of %d KV heads are too many for one call", p.tokens, p.nkv);
    const dim3 grid(static_cast<unsigned>(ctas) + 1);
    if (p.hd == 64) return d->launch(kv_q8_store_kernel<T, 64>, grid, dim3(threads), 0, p, rows);
    return d->launch(kv_q8_store_kernel<T, 128>, grid, dim3(threads), 0, p, rows);
}

template <typename T>
l0b_status load_as(l0b_device* d, const KvQ8Params& p) {
    return d->launch(kv_q8_load_kernel<T>, dim3((p.tokens + 7) / 8 + 1), dim3(256), 0, p);
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
