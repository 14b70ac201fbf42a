// Causal attention over packed sequences with f32 queries, at about f32 accuracy (sm_100a, mma.sync m16n8k16, f32
// accumulators). 16-bit queries take attention_packed.cu.
//
// A CTA takes 64 query rows of one head (four warps of 16) and walks its keys 64 at a time, K and V double-buffered by
// cp.async in swizzled shared memory. Queries and weights enter the MMA as sums of 16-bit terms of the keys' type: two
// f16 terms (22 bits) or three bf16 terms (24 bits); each query row is first scaled by a power of two, and weights
// carry 2^14, so that the small terms stay normal f16 numbers. The MMA truncates its sums, so O takes each tile's
// P V from accumulators of its own by an f32 add: four steps a sum, not one for every 16 keys of the sequence.
//
// 64-row blocks of sequence i sit at slots floor(q_starts[i] / 64) + i and on, which leaves room for each sequence's
// blocks without a prefix sum; a slot with no rows ends at once. Late slots first: they see the most keys.
//
// Values that the mask hides reach no row, whatever they hold: key rows behind the sequence are read as zeros, and in
// a tile that some row sees in part, value rows with an infinity or a NaN are set aside and added, where seen, at the
// end.
//
// Bound by mma.sync (a quarter of tcgen05's rate, two or three products for one) for long sequences.
#include <mutex>

#include "ops.cuh"
#include "packed.cuh"
#include "packed_attn.cuh"
#include "tma.cuh"

namespace l0b {

namespace {

constexpr int kB = 64;             // query rows, and keys of a tile
constexpr float kWeightBits = 14.f;  // weights are at most 2^14

template <typename T> constexpr int kTerms = DT<T>::id == L0B_F16 ? 2 : 3;

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT<T>::id == L0B_F16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool TRANS>
__device__ __forceinline__ void load_4x8x8(uint32_t (&r)[4], uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    return DT<T>::id == L0B_F16 ? half2_bits_to_float2(w) : bf162_bits_to_float2(w);
}

// (a, b) as a sum of kTerms<T> pairs of 16-bit values.
template <typename T>
__device__ __forceinline__ void split(float a, float b, uint32_t (&term)[kTerms<T>]) {
#pragma unroll
    for (int i = 0; i < kTerms<T>; ++i) {
        term[i] = pack2<T>(a, b);
        const float2 f = unpack2<T>(term[i]);
        a -= f.x;
        b -= f.y;
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(128, 2) packed_f32_kernel(const PackedAttnParams p) {
    constexpr int NT = kTerms<T>, RB = HD * 2, TILE = kB * RB;  // terms, bytes of a row, of a tile
    constexpr int KS = HD / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* q_s = smem;                // [NT][kB][HD]
    uint8_t* kv_s = smem + NT * TILE;   // [2 stages][K, V][kB][HD]
    __shared__ float factor_s[kB];
    __shared__ uint32_t bad_s[2][2];    // [cut tile][64 keys]: value rows set aside
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();

    // Sequence and block of this CTA's slot.
    const int head = blockIdx.x % p.nh, slots = p.tokens / kB + p.count, slot = slots - 1 - blockIdx.x / p.nh;
    int seq = -1;
    for (int i0 = 0; i0 < p.count; i0 += 128) {
        const int i = i0 + tid;
        seq += __syncthreads_count(i < p.count && max(__ldg(p.q_starts + i), 0) / kB + i <= slot);
    }
    if (seq < 0) return;
    const PackedSeq s = packed_seq(p, seq);
    const int tok = (slot - (s.q0 / kB + seq)) * kB, rows = min(kB, s.n - tok);
    if (tid == 0 && tok == 0 &&
        (__ldg(p.q_starts + seq) < 0 || __ldg(p.q_starts + seq + 1) > p.tokens || __ldg(p.kv_starts + seq) < 0 ||
         __ldg(p.kv_starts + seq + 1) > p.kv_tokens || __ldg(p.q_starts + seq) > __ldg(p.q_starts + seq + 1) ||
         __ldg(p.kv_starts + seq) > __ldg(p.kv_starts + seq + 1)))
        flag_bad_index(p.error);
    if (tok < 0 || rows <= 0) return;
    const int first = s.m - s.n + tok, last = first + rows - 1;  // the last key that the first and last row see
    const int tiles = last >= 0 ? last / kB + 1 : 0, full = min(tiles, max(0, first + 1) / kB);
    const int kvh = head / (p.nh / p.nkv);
    const T* k = static_cast<const T*>(p.k) + static_cast<long long>(s.k0) * p.k_stride + kvh * HD;
    const T* v = static_cast<const T*>(p.v) + static_cast<long long>(s.k0) * p.v_stride + kvh * HD;

    auto load = [&](int j, int st) {
        uint8_t* dst = kv_s + st * 2 * TILE;
#pragma unroll 4
        for (int e = tid; e < kB * (HD / 8); e += 128) {
            const int r = e / (HD / 8), c = e % (HD / 8), key = j * kB + r;
            const uint32_t at = smem_addr(dst) + r * RB + ((c ^ (r & 7)) << 4);
            const int bytes = key < s.m ? 16 : 0;  // 0: zeros, nothing read
            const long long row = key < s.m ? key : 0;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(k + row * p.k_stride + c * 8), "r"(bytes) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + TILE), "l"(v + row * p.v_stride + c * 8), "r"(bytes)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (tiles > 0) load(0, 0);

    // Query terms: a warp's own 16 rows, eight rows' loads in flight, a row spread over the lanes.
    if (tid < 4) bad_s[tid >> 1][tid & 1] = 0;
    for (int r0 = 0; r0 < 16; r0 += 8) {
        float x[8][HD / 32];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const float* q = static_cast<const float*>(p.q) +
                             static_cast<long long>(s.q0 + tok + min(warp * 16 + r0 + r, rows - 1)) * p.q_stride +
                             static_cast<long long>(head) * HD + lane * (HD / 32);
            if constexpr (HD == 128) {
                const float4 y = __ldg(reinterpret_cast<const float4*>(q));
                x[r][0] = y.x; x[r][1] = y.y; x[r][2] = y.z; x[r][3] = y.w;
            } else {
                const float2 y = __ldg(reinterpret_cast<const float2*>(q));
                x[r][0] = y.x; x[r][1] = y.y;
            }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int row = warp * 16 + r0 + r;
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) top = fmaxf(top, fabsf(x[r][i]));
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
            const int bits = top > 0.f && top < __int_as_float(0x7F800000) ? min(13 - ilogbf(top), 126) : 0;  // to [2^13, 2^14)
            const float up = ldexpf(1.f, bits);
            if (lane == 0) factor_s[row] = ldexpf(p.scale * 1.44269504088896341f, -bits);
#pragma unroll
            for (int i = 0; i < HD / 32; i += 2) {
                uint32_t term[NT];
                split<T>(x[r][i] * up, x[r][i + 1] * up, term);
                const int d = lane * (HD / 32) + i;  // dim
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    *reinterpret_cast<uint32_t*>(q_s + n * TILE + row * RB + (((d >> 3) ^ (row & 7)) << 4) + (d & 7) * 2) = term[n];
            }
        }
    }
    __syncwarp();
    float f[2], m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
    int limit[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f[h] = factor_s[warp * 16 + g + 8 * h];
        limit[h] = first + warp * 16 + g + 8 * h;
    }
    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    for (int j = 0; j < tiles; ++j) {
        const int st = j & 1;
        uint8_t* kt = kv_s + st * 2 * TILE;
        uint8_t* vt = kt + TILE;
        if (j + 1 < tiles) {
            load(j + 1, st ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        if (j >= full) {
            for (int e = tid; e < kB * (HD / 8); e += 128) {
                const int r = e / (HD / 8);
                const uint4 w = *reinterpret_cast<const uint4*>(vt + e * 16);
                if (not_finite<DT<T>::id == L0B_BF16>(w)) atomicOr(&bad_s[j - full][r >> 5], 1u << (r & 31));
            }
            __syncthreads();
            const uint32_t bad[2] = {bad_s[j - full][0], bad_s[j - full][1]};
            if (bad[0] | bad[1]) {
                for (int e = tid; e < kB * (HD / 8); e += 128) {
                    const int r = e / (HD / 8);
                    if ((bad[r >> 5] >> (r & 31)) & 1) *reinterpret_cast<uint4*>(vt + e * 16) = make_uint4(0, 0, 0, 0);
                }
            }
            __syncthreads();
        }
        float sc[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            uint32_t a[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int r = warp * 16 + (lane & 15), c = 2 * kk + (lane >> 4);
                load_4x8x8<false>(a[i], smem_addr(q_s) + i * TILE + r * RB + ((c ^ (r & 7)) << 4));
            }
            uint32_t b[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int r = n * 16 + (lane & 7) + ((lane >> 4) << 3), c = 2 * kk + ((lane >> 3) & 1);
                load_4x8x8<false>(b[n], smem_addr(kt) + r * RB + ((c ^ (r & 7)) << 4));
            }
            // small terms first; eight sums in turn, so that no MMA waits for the one before it
#pragma unroll
            for (int i = NT - 1; i >= 0; --i) {
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    mma<T>(sc[2 * n], a[i], b[n][0], b[n][1]);
                    mma<T>(sc[2 * n + 1], a[i], b[n][2], b[n][3]);
                }
            }
        }
        float keep[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = kNegInf;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = sc[n][2 * h + e];
                    x *= f[h];
                    if (j >= full && j * kB + n * 8 + 2 * t + e > limit[h]) x = kNegInf;
                    top = fmaxf(top, x);
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[h], top), shift = now == kNegInf ? 0.f : now - kWeightBits;
            keep[h] = now == m[h] ? 1.f : exp2_fast(m[h] - now);
            m[h] = now;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                sc[n][2 * h] = exp2_fast(sc[n][2 * h] - shift);
                sc[n][2 * h + 1] = exp2_fast(sc[n][2 * h + 1] - shift);
                sum += sc[n][2 * h] + sc[n][2 * h + 1];
            }
            l[h] = fmaf(l[h], keep[h], sum);
        }
        uint32_t w[4][NT][4];  // weights of 16 keys a step, as A operands
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float* x = sc[2 * kk + (q >> 1)] + 2 * (q & 1);
                uint32_t term[NT];
                split<T>(x[0], x[1], term);
#pragma unroll
                for (int i = 0; i < NT; ++i) w[kk][i][q] = term[i];
            }
        }
#pragma unroll
        for (int n = 0; n < HD / 8; n += 8) {
            float acc[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint32_t b[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = 16 * kk + (lane & 15), c = n + 2 * q + (lane >> 4);
                    load_4x8x8<true>(b[q], smem_addr(vt) + r * RB + ((c ^ (r & 7)) << 4));
                }
#pragma unroll
                for (int i = NT - 1; i >= 0; --i) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        mma<T>(acc[2 * q], w[kk][i], b[q][0], b[q][1]);
                        mma<T>(acc[2 * q + 1], w[kk][i], b[q][2], b[q][3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[n + i][0] = fmaf(o[n + i][0], keep[0], acc[i][0]);
                o[n + i][1] = fmaf(o[n + i][1], keep[0], acc[i][1]);
                o[n + i][2] = fmaf(o[n + i][2], keep[1], acc[i][2]);
                o[n + i][3] = fmaf(o[n + i][3], keep[1], acc[i][3]);
            }
        }
        __syncthreads();  // the stage is filled again
    }

#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int row = warp * 16 + g + 8 * h;
        if (row >= rows) continue;
        for (int j = full; j < tiles; ++j) {
            for (int q = 0; q < 2; ++q) {
                for (uint32_t bits = bad_s[j - full][q]; bits; bits &= bits - 1) {
                    const int key = j * kB + q * 32 + __ffs(bits) - 1;
                    if (key > limit[h]) break;
                    const float c = p.scale * 1.44269504088896341f;
                    const float x = weight_anew<T, HD>(p, s, head, tok + row, key, c, m[h] - kWeightBits);
                    const T* at = v + key * p.v_stride + 2 * t;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                        o[n][2 * h] = fmaf(x, load_as_float(at, DT<T>::id, n * 8), o[n][2 * h]);
                        o[n][2 * h + 1] = fmaf(x, load_as_float(at, DT<T>::id, n * 8 + 1), o[n][2 * h + 1]);
                    }
                }
            }
        }
        const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
        float* out = static_cast<float*>(p.out) + static_cast<long long>(s.q0 + tok + row) * p.out_stride +
                     static_cast<long long>(head) * HD + 2 * t;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
            *reinterpret_cast<float2*>(out + n * 8) = make_float2(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
    }
}

template <typename T, int HD>
l0b_status launch(l0b_device* d, const PackedAttnParams& p) {
    auto kernel = packed_f32_kernel<T, HD>;
    constexpr size_t smem = static_cast<size_t>(kTerms<T> + 4) * kB * HD * 2;
    {
        static bool configured[64] = {};
        static std::mutex mu;
        std::lock_guard<std::mutex> lock(mu);
        if (d->index >= 64 || !configured[d->index]) {
            L0B_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
            if (d->index < 64) configured[d->index] = true;
        }
    }
    const long long grid = (static_cast<long long>(p.tokens) / kB + p.count) * p.nh;
    L0B_REQUIRE(grid <= INT32_MAX, L0B_ERR_OUT_OF_RANGE, "%d rows of %d heads are too many for one call", p.tokens, p.nh);
    return d->launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(128), smem, p);
}

}  // namespace

l0b_status k_attention_packed_f32(l0b_suite*, l0b_device* d, const PackedAttnParams& p) {
    if (p.kv_dtype == L0B_F16) return p.hd == 64 ? launch<__half, 64>(d, p) : launch<__half, 128>(d, p);
    return p.hd == 64 ? launch<__nv_bfloat16, 64>(d, p) : launch<__nv_bfloat16, 128>(d, p);
}

}  // namespace l0b
