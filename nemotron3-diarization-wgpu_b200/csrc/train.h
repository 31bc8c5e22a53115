// Internal interfaces of the training operators (rope.cu, residual_norm.cu,
// attention_train.cu, attention_train_tc.cu, train_api.cpp).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/n3d.h"
#include "n3d_internal.h"

namespace n3d {

// An n3d_heads on the device side: pointer and strides, in elements.
struct HeadsView {
    void* p;
    long long seq, row, head;
};

inline int dtype_size(int dtype) { return dtype == N3D_F32 ? 4 : 2; }

// ---- rope.cu
struct RopeArgs {
    HeadsView x[2], y[2];
    int heads0, heads;         // heads of tensor 0, and of both
    int rows;                  // rows of a sequence
    long long tokens;          // seqs * rows
    const int32_t* positions;  // [tokens] or null
    long long first;
    int head_dim, rotary_dim;
    float factor;
    int transpose;
    int in_place[2];
};
void launch_rope(cudaStream_t s, const RopeArgs& a, const n3d_rope_plan& plan, int dtype);

}  // namespace n3d
