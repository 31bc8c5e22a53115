// fp32 operands of the training attention for the tensor cores: the largest magnitude of
// q, k, v (and dout), then each as two fp16 arrays of x s (h = x s rounded to 11 bits, l the
// rest; s the power of two that brings the largest magnitude to at most 2^15), as the
// library's other fp32 products (n3d_device.cuh).  Rows past the lengths become zeros.
//
// For the gradient the same pass takes, per query row, -lse log2 e, -D = -(dout . out) and
// |dout row|, in fp32 from the unsplit tensors, and the largest |dout row| of each head.
//
// Bound: memory, two reads of each operand and one write of the same size.  Two launches
// in front of one or two that compute on 64 rows x 64 columns x head_dim per 12 KB read.

#include <cuda_fp16.h>

#include <algorithm>

#include "n3d_device.cuh"
#include "train.h"

namespace n3d {

namespace {

constexpr int THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f;

struct Operand {
    HeadsView t;
    const int32_t* len;
    int rows, heads;
    long long lines;  // seqs * heads * rows
    __half* out;      // part 0; part 1 lies lines * head_dim further
};
struct SplitArgs {
    Operand op[4];  // q, k, v, dout
    HeadsView o;
    const float* lse;
    AttnSplitSpace sp;
    long long heads_total;  // seqs * q_heads
    int q_tiles, backward;
};

// Line i of an operand: sequence, head, row; whether the row is inside its length.
struct Line {
    long long seq;
    int head, row;
    bool live;
};
__device__ __forceinline__ Line line_of(const Operand& p, long long i) {
    Line l;
    const long long sh = i / p.rows;
    l.row = (int)(i - sh * p.rows);
    l.seq = sh / p.heads;
    l.head = (int)(sh - l.seq * p.heads);
    l.live = !p.len || l.row < p.len[l.seq];
    return l;
}
__device__ __forceinline__ const float* line_ptr(const HeadsView& t, const Line& l) {
    return static_cast<const float*>(t.p) + l.seq * t.seq + (long long)l.row * t.row + l.head * t.head;
}

// blockIdx.y: the operand.  A warp per line.  Infinities and NaN do not count: they make
// their own products NaN whatever the scale.
template <int PER>  // elements of a lane: head_dim / 32
__global__ void __launch_bounds__(THREADS) attention_absmax_kernel(const __grid_constant__ SplitArgs a) {
    __shared__ float part[THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const Operand& p = a.op[blockIdx.y];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (a.backward && blockIdx.y == 3)
        for (long long i = blockIdx.x * THREADS + threadIdx.x; i < a.heads_total; i += gridDim.x * THREADS)
            a.sp.head_norm[i] = 0.0f;
    float m = 0.0f;
    for (long long i = blockIdx.x * (THREADS / 32) + warp; i < p.lines; i += gridDim.x * (THREADS / 32)) {
        const Line l = line_of(p, i);
        if (!l.live) continue;
        const float* x = line_ptr(p.t, l);
#pragma unroll
        for (int c = 0; c < PER; c++) {
            const float v = fabsf(x[lane + 32 * c]);
            if (v < INFINITY) m = fmaxf(m, v);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) part[warp] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < THREADS / 32; i++) m = fmaxf(m, part[i]);
        a.sp.partial[blockIdx.y * kSplitBlocks + blockIdx.x] = m;
    }
}

template <int PER>
__global__ void __launch_bounds__(THREADS) attention_split_kernel(const __grid_constant__ SplitArgs a) {
    __shared__ float part[THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const Operand& p = a.op[blockIdx.y];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = 0.0f;
    for (int i = threadIdx.x; i < kSplitBlocks; i += THREADS) m = fmaxf(m, a.sp.partial[blockIdx.y * kSplitBlocks + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) part[warp] = m;
    __syncthreads();
    m = part[0];
    for (int i = 1; i < THREADS / 32; i++) m = fmaxf(m, part[i]);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.sp.maxima[blockIdx.y] = m;
    const float s = split_scale_of(m);
    for (long long i = blockIdx.x * (THREADS / 32) + warp; i < p.lines; i += gridDim.x * (THREADS / 32)) {
        const Line l = line_of(p, i);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (l.live) {
            const float* x = line_ptr(p.t, l) + lane * PER;
#pragma unroll
            for (int c = 0; c < PER; c++) v[c] = x[c];
        }
        uint32_t h[2], lo[2];
        split2x2(v[0], v[1], s, h[0], lo[0]);
        split2x2(v[2], v[3], s, h[1], lo[1]);
        __half* out = p.out + i * 32 * PER + lane * PER;
        __half* low = out + p.lines * 32 * PER;
        if (PER == 2) {
            *reinterpret_cast<uint32_t*>(out) = h[0];
            *reinterpret_cast<uint32_t*>(low) = lo[0];
        } else {
            *reinterpret_cast<uint2*>(out) = make_uint2(h[0], h[1]);
            *reinterpret_cast<uint2*>(low) = make_uint2(lo[0], lo[1]);
        }
        if (a.backward && blockIdx.y == 3) {
            float dot = 0.0f, norm2 = 0.0f;
            if (l.live) {
                const float* o = line_ptr(a.o, l) + lane * PER;
#pragma unroll
                for (int c = 0; c < PER; c++) dot += v[c] * o[c], norm2 += v[c] * v[c];
            }
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) {
                dot += __shfl_xor_sync(0xffffffffu, dot, k);
                norm2 += __shfl_xor_sync(0xffffffffu, norm2, k);
            }
            if (lane == 0) {
                const long long sqh = l.seq * p.heads + l.head;
                float* st = a.sp.stats + (sqh * a.q_tiles * 2 + l.row / 64) * kSplitStat + l.row % 64;
                const float lse = l.live ? a.lse[sqh * p.rows + l.row] : -INFINITY;
                st[0] = lse == -INFINITY ? -INFINITY : -lse * LOG2E;
                st[64] = -dot;
                st[128] = sqrtf(norm2);
                // a maximum of non-negative floats, the same in any order
                if (norm2 > 0.0f) atomicMax(reinterpret_cast<int*>(a.sp.head_norm + sqh), __float_as_int(sqrtf(norm2)));
                // the rows of the last block of 64 that do not exist belong to it too
                if (l.row == p.rows - 1)
                    for (int r = p.rows; r % 64 != 0; r++) {
                        float* e = a.sp.stats + (sqh * a.q_tiles * 2 + r / 64) * kSplitStat + r % 64;
                        e[0] = -INFINITY;
                        e[64] = 0.0f;
                        e[128] = 0.0f;
                    }
            }
        }
    }
}

}  // namespace

size_t attn_split_space(void* base, size_t seqs, size_t q_heads, size_t k_heads, size_t q_rows, size_t k_rows,
                        size_t head_dim, bool backward, AttnSplitSpace* out) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        void* p = static_cast<char*>(base) + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    AttnSplitSpace s{};
    const size_t q = seqs * q_heads * q_rows * head_dim * 4, k = seqs * k_heads * k_rows * head_dim * 4;
    s.maxima = static_cast<float*>(take(4 * sizeof(float)));
    s.partial = static_cast<float*>(take(4 * kSplitBlocks * sizeof(float)));
    s.q = take(q);
    s.k = take(k);
    s.v = take(k);
    if (backward) {
        s.dout = take(q);
        s.head_norm = static_cast<float*>(take(seqs * q_heads * sizeof(float)));
        s.stats = static_cast<float*>(take(seqs * q_heads * ((q_rows + 127) / 128) * 2 * kSplitStat * sizeof(float)));
    }
    if (out) *out = s;
    return at;
}

void launch_attention_split(cudaStream_t s, const AttnArgs& a, const AttnSplitSpace& sp, bool backward) {
    SplitArgs t{};
    const HeadsView views[4] = {a.q, a.k, a.v, a.dout};
    void* const outs[4] = {sp.q, sp.k, sp.v, sp.dout};
    for (int i = 0; i < (backward ? 4 : 3); i++) {
        const bool keys = i == 1 || i == 2;
        Operand& p = t.op[i];
        p.t = views[i];
        p.len = keys ? a.k_len : a.q_len;
        p.rows = keys ? a.k_rows : a.q_rows;
        p.heads = keys ? a.k_heads : a.q_heads;
        p.lines = (long long)a.seqs * p.heads * p.rows;
        p.out = static_cast<__half*>(outs[i]);
    }
    t.o = a.o;
    t.lse = a.lse;
    t.sp = sp;
    t.heads_total = (long long)a.seqs * a.q_heads;
    t.q_tiles = (a.q_rows + 127) / 128;
    t.backward = backward;
    const dim3 grid(kSplitBlocks, backward ? 4 : 3);
    if (a.head_dim == 64) {
        launch_pdl(attention_absmax_kernel<2>, grid, dim3(THREADS), 0, s, t);
        launch_pdl(attention_split_kernel<2>, grid, dim3(THREADS), 0, s, t);
    } else {
        launch_pdl(attention_absmax_kernel<4>, grid, dim3(THREADS), 0, s, t);
        launch_pdl(attention_split_kernel<4>, grid, dim3(THREADS), 0, s, t);
    }
}

}  // namespace n3d
