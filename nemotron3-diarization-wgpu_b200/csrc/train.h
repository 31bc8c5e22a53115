// Internal interfaces of the training operators (rope.cu, residual_norm.cu,
// attention_train.cu, attention_train_tc.cu, train_api.cpp).
#pragma once

#include <cuda_runtime.h>

#include <climits>
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

// ---- residual_norm.cu, residual_norm_grad.cu
struct ResidualArgs {
    long long rows;
    int cols;
    int post, pre;  // n3d_norm
    float post_eps, pre_eps, scale;
    long long rows_per_gate;  // 0: no gate
    const float *post_w, *post_b, *gate, *pre_w, *pre_b;
    const void *x, *block, *r, *dy, *dr;
    long long ld_x, ld_block, ld_r, ld_dy, ld_dr;
    void *r_out, *y, *dx, *dblock;
    long long ld_r_out, ld_y, ld_dx, ld_dblock;
    float *dgate, *dpost_w, *dpost_b, *dpre_w, *dpre_b;
    float* sums;        // [blocks][4][cols]: post weight and bias, pre weight and bias
    float* gate_parts;  // [slots][2][cols]
    int slots;          // row ranges of the gradient kernel
    int wide;           // every row and weight starts on four whole elements, as do the row strides and cols
};
void launch_residual_norm(cudaStream_t s, const ResidualArgs& a, int residual_dtype, int block_dtype);
// How the gradient kernel splits the rows: `slots` ranges (range i is rows
// rows * i / slots ..), `blocks` thread blocks, `threads` per row.
struct ResidualSplit {
    int threads, per_block, slots, blocks;
};
ResidualSplit residual_split(long long rows, int cols, bool wide);
void launch_residual_norm_grad(cudaStream_t s, const ResidualArgs& a, int residual_dtype, int block_dtype);

// ---- attention_train.cu, attention_train_tc.cu
struct AttnArgs {
    HeadsView q, k, v, o, dout, dq, dk, dv;
    float* lse;         // [seqs, q_heads, q_rows], null: not wanted (forward)
    float* row_dot;     // the workspace
    int* err;           // where an expired wait records its site
    int seqs, q_rows, k_rows, q_heads, k_heads, head_dim;
    float scale;
    int left, right, offset;      // kNoLimit where unlimited
    const int32_t *q_len, *k_len;  // null: all rows
};
constexpr int kNoLimit = INT_MAX;
constexpr int kMaxReach = 1 << 30;  // of left, right and offset: their sums stay inside 32 bits where that matters

// The rows of one sequence and which keys a query row sees.
struct AttnMask {
    int q_len, k_len, left, right, offset;
#ifdef __CUDACC__
    __device__ __forceinline__ AttnMask(const AttnArgs& a, int seq)
        : q_len(a.q_len ? min(max(a.q_len[seq], 0), a.q_rows) : a.q_rows),
          k_len(a.k_len ? min(max(a.k_len[seq], 0), a.k_rows) : a.k_rows),
          left(a.left),
          right(a.right),
          offset(a.offset) {}
    // the same of a sequence whose row and column lengths are known (`by_key`: rows are keys)
    __device__ __forceinline__ AttnMask(const AttnArgs& a, int, int row_len, int col_len, bool by_key)
        : q_len(by_key ? col_len : row_len),
          k_len(by_key ? row_len : col_len),
          left(a.left),
          right(a.right),
          offset(a.offset) {}
    // key rows [first, last) of query row i, empty when last <= first
    __device__ __forceinline__ int first_key(int i) const {
        return left >= kNoLimit ? 0 : (int)max(0LL, (long long)i + offset - left);
    }
    __device__ __forceinline__ int last_key(int i) const {
        return right >= kNoLimit ? k_len : (int)max(0LL, min((long long)k_len, (long long)i + offset + right + 1));
    }
    // query rows [first, last) that see key row j
    __device__ __forceinline__ int first_query(int j) const {
        return right >= kNoLimit ? 0 : (int)max(0LL, (long long)j - offset - right);
    }
    __device__ __forceinline__ int last_query(int j) const {
        return left >= kNoLimit ? q_len : (int)max(0LL, min((long long)q_len, (long long)j - offset + left + 1));
    }
#endif
};
// Workspace of the gradient of 16-bit tensors, in floats: on the fp32 units dout . out of each
// row; on the tensor cores two blocks of 128 for every 128 query rows of a head (row
// statistics of 64 rows each) and one (the largest |dout row| of the 128).
inline size_t attn_workspace_floats(size_t seqs, size_t q_heads, size_t q_rows) {
    return seqs * q_heads * ((q_rows + 127) / 128) * (2 * 128 + 1);
}
// Workspace of fp32 tensors on the tensor cores (attention_train_split.cu): what belongs to
// each row, and each operand as two fp16 arrays [part][seqs][heads][rows][hd].
constexpr int kSplitStat = 256;  // floats per 64 query rows: -lse log2 e | -D | unit of q | unit of dout
constexpr int kKeyStat = 128;    // floats per 64 key rows: unit of k | unit of v
struct AttnSplitSpace {
    float* stats;      // [seqs * q_heads][q tiles of 128][2][kSplitStat]
    float* key_stats;  // [seqs * k_heads][k tiles of 64][kKeyStat]
    void *q, *k, *v, *dout;
};
// Lays the workspace out at `base` (may be null) and returns its size in bytes.
size_t attn_split_space(void* base, size_t seqs, size_t q_heads, size_t k_heads, size_t q_rows, size_t k_rows,
                        size_t head_dim, bool backward, AttnSplitSpace* out);
void launch_attention_split(cudaStream_t s, const AttnArgs& a, const AttnSplitSpace& sp, bool backward);
// attention_train_tc.cu: whether the call's tensors fit TMA (16-bit types, whole 16-byte
// words, no broadcast dimension), and the launches; fp32 tensors go through the split.
bool attention_tc_fits(const AttnArgs& a, int dtype, bool backward);
void launch_attention_train_tc(cudaStream_t s, const AttnArgs& a, int dtype, bool backward);
// Whether fp32 tensors of these sizes are split for the tensor cores.
bool attention_split_pays(size_t q_rows, size_t k_rows, bool backward);
void launch_attention_forward(cudaStream_t s, const AttnArgs& a, int dtype);
void launch_attention_backward(cudaStream_t s, const AttnArgs& a, int dtype);

}  // namespace n3d
