// Device helpers of the ops over packed sequences (attention_packed.cu, attention_q8.cu, kv_q8.cu).
//
// What these ops read - rows, codes, scales, starts, positions, lengths - may come from the kernel just before, and under
// programmatic dependent launch that kernel still runs while this one starts. So nothing of it is read through the
// read-only path (ld.global.nc), which asks that memory stays as it is for a kernel's whole life; pdl_wait orders the
// ordinary loads behind it.
#pragma once

#include "common.cuh"

namespace l0b {

// A start, position or length read on the device lay outside its buffers (l0b_device_error_status, bit 1).
__device__ __forceinline__ void flag_bad_index(int* error) {
    if (error) atomicOr(error, 2);
}

// A start read on the device, kept within [0, rows]: differences of two of them cannot overflow.
__device__ __forceinline__ int clamp_start(int start, int rows) { return max(0, min(start, rows)); }

// Index of the last of starts[0, count) that is <= t, -1 if none: the sequence of packed row t when
// t < starts[index + 1] (an empty sequence shares its start with the next and is passed over). All threads
// of the CTA call it together and get the same answer; every start is read at once, so the latency is one
// load for up to blockDim.x sequences, where a binary search would wait for log2(count) of them in turn.
__device__ __forceinline__ int block_find_sequence(const int* starts, int count, int t) {
    int n = 0;
    for (int i0 = 0; i0 < count; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        n += __syncthreads_count(i < count && starts[i] <= t);
    }
    return n - 1;
}

// 16 bytes that are read once: no L1 allocation.
__device__ __forceinline__ uint4 ld_once_v4(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

// Eight consecutive elements of f32 / f16 / bf16 as f32; p on 16 bytes.
template <typename T>
__device__ __forceinline__ void load8_f32(const T* p, float (&o)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = DT<T>::id == L0B_F16 ? half2_bits_to_float2(w[i]) : bf162_bits_to_float2(w[i]);
            o[2 * i] = f.x;
            o[2 * i + 1] = f.y;
        }
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT<T>::id == L0B_F16) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Eight f32 values to eight consecutive elements, each rounded once; p on 16 bytes.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}

}  // namespace l0b
