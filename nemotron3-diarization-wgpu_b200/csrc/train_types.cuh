// Element types of the training operators: 16-byte vectors of fp32, bf16 and fp16, held
// as fp32 in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace n3d {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
    return __half2float(v);
}
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}

// Two values rounded to T, a in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <class T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack_pair<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
}

// N consecutive elements as raw words, loaded and stored in words of 8 bytes (four 16-bit
// elements) or 16 (N elements must fill whole words and p must be aligned to them), or one
// element (N = 1).
template <class T, int N>
struct Vec {
    using W = typename std::conditional<N * sizeof(T) == 8, uint2, uint4>::type;
    static constexpr int WORDS = N * (int)sizeof(T) / (int)sizeof(W);
    W w[WORDS];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = __ldg(reinterpret_cast<const W*>(p) + i);
    }
    // for data that the same kernel writes (in-place calls): no read-only path
    __device__ __forceinline__ void load_rw(const T* p) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = *(reinterpret_cast<const W*>(p) + i);
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < WORDS; i++) reinterpret_cast<W*>(p)[i] = w[i];
    }
    __device__ __forceinline__ void get(float* f) const {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) f[i] = __uint_as_float(u[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const float2 t = unpack_pair<T>(u[i]);
                f[2 * i] = t.x, f[2 * i + 1] = t.y;
            }
        }
    }
    __device__ __forceinline__ void set(const float* f) {
        uint32_t* u = reinterpret_cast<uint32_t*>(w);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) u[i] = __float_as_uint(f[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; i++) u[i] = pack_pair<T>(f[2 * i], f[2 * i + 1]);
        }
    }
};
template <class T>
struct Vec<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void load_rw(const T* p) { v = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ void get(float* f) const { f[0] = to_f32<T>(v); }
    __device__ __forceinline__ void set(const float* f) { v = from_f32<T>(f[0]); }
};

}  // namespace n3d
