// Shared by the residual-norm kernels: rows spread over TPR threads, sums over a row.
#pragma once

#include "n3d_device.cuh"
#include "train.h"
#include "train_types.cuh"

namespace n3d {

// Columns of thread t of a row: EPT of them, in chunks of VEC consecutive ones; chunk k
// starts at (k * TPR + t) * VEC, so that a warp's chunk is one run of memory.  VEC is 4:
// one 16-byte load of fp32 (a weight, a residual), one 8-byte load of 16 bits.  (With 8, a
// warp's fp32 loads covered every other 16 bytes of 1 KB and took twice the L1 wavefronts,
// which bound the kernels: forward of 8191 x 4096 in bf16 73 us.)
template <int VEC, int TPR>
__device__ __forceinline__ int chunk_col(int k, int t) {
    return (k * TPR + t) * VEC;
}

// VEC fp32 values (weights), or `other` for a null pointer.
template <int VEC>
__device__ __forceinline__ void load_weights(const float* p, int col, float other, float* v) {
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = other;
        return;
    }
    if constexpr (VEC == 1) {
        v[0] = __ldg(p + col);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(p + col + i));
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
    }
}

// Sums of NV values over the TPR threads of a row, the same in every thread and taken in
// a fixed order.  In a warp the values are first dealt out: each exchange halves the
// values a lane holds (8 values take 4 + 2 + 1 shuffles and two more, instead of 40), until
// GS lanes share one value; the warps' sums meet in `buf` (one per call site of a row,
// TPR / 32 * NV floats, which may be written again once a later sum of the row has been
// taken).  Threads of a row wait only for one another (named barrier 1 + slot of the block).
template <int TPR, int NV>
__device__ __forceinline__ void row_sums(float (&v)[NV], float* buf, int slot) {
    constexpr int P = NV == 1 ? 1 : NV == 2 ? 2 : NV <= 4 ? 4 : 8, GS = 32 / P;
    static_assert(NV <= 8, "at most 8 values");
    const int lane = threadIdx.x & 31, q = lane / GS;  // the value of this lane
    float x[P];
#pragma unroll
    for (int i = 0; i < P; i++) x[i] = i < NV ? v[i] : 0.0f;
#pragma unroll
    for (int n = P / 2, o = 16; n > 0; n /= 2, o /= 2)
#pragma unroll
        for (int i = 0; i < n; i++) {
            const bool up = lane & o;
            const float keep = up ? x[n + i] : x[i], send = up ? x[i] : x[n + i];
            x[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    float z = x[0];
#pragma unroll
    for (int o = GS / 2; o > 0; o /= 2) z += __shfl_xor_sync(0xffffffffu, z, o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        const int warp = (threadIdx.x % TPR) >> 5, i = lane % GS;
        if (i == 0 && q < NV) buf[q * W + warp] = z;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "n"(TPR) : "memory");
        z = 0.0f;
        if (q < NV) {
            if constexpr (W > GS) {
#pragma unroll
                for (int j = 0; j < W / GS; j++) z += buf[q * W + i * (W / GS) + j];
            } else if (i < W) {
                z = buf[q * W + i];
            }
        }
#pragma unroll
        for (int o = GS / 2; o > 0; o /= 2) z += __shfl_xor_sync(0xffffffffu, z, o);
    }
#pragma unroll
    for (int i = 0; i < NV; i++) v[i] = NV == 1 ? z : __shfl_sync(0xffffffffu, z, i * GS);
}

}  // namespace n3d
