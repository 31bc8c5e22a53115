// fp32 operands of the training attention for the tensor cores: the largest magnitude of
// q, k, v (and dout), then each as two fp16 arrays of x s (h = x s rounded to 11 bits, l the
// rest; s the power of two that brings the largest magnitude to at most 2^15), as the
// library's other fp32 products (n3d_device.cuh).  Rows past the lengths become zeros.
//
// For the gradient the same pass takes, per query row, -lse log2 e, -D = -(dout . out) and
// |dout row|, in fp32 from the unsplit tensors, and the largest |dout row| of each head.
//
// Bound: latency (four lines of a thread are in flight) before memory: two reads of each
// operand and one write of the same size.  Measured on a B200, cold: q, k and v of 8 x 501 rows,
// 8 heads of 64 (25 MB) 13 us for the magnitudes and 16 us for the split; with dout and the
// statistics 16 and 22 us.

#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "n3d_device.cuh"
#include "train.h"

namespace n3d {

namespace {

constexpr int THREADS = 256;
constexpr int ILP = 4;  // lines of a thread in flight
constexpr float LOG2E = 1.4426950408889634f;

struct Operand {
    HeadsView t;
    const int32_t* len;
    int rows, heads;
    int lines;    // seqs * heads * rows
    int wide;     // every line starts on 16 bytes
    __half* out;  // part 0; part 1 lies lines * head_dim further
};
struct SplitArgs {
    Operand op[4];  // q, k, v, dout
    HeadsView o;
    int o_wide;
    const float* lse;
    AttnSplitSpace sp;
    int heads_total;  // seqs * q_heads
    int q_tiles, backward;
};

// Line i of an operand: sequence * heads + head, sequence, row; whether the row is inside its length.
struct Line {
    int sh, seq, row;
    bool live;
};
__device__ __forceinline__ Line line_of(const Operand& p, int i) {
    Line l;
    l.sh = i / p.rows;
    l.row = i - l.sh * p.rows;
    l.seq = l.sh / p.heads;
    l.live = !p.len || l.row < p.len[l.seq];
    return l;
}
// Four consecutive elements of a line from c on.
__device__ __forceinline__ float4 line_load(const HeadsView& t, const Line& l, int heads, int c, bool wide) {
    const float* x = static_cast<const float*>(t.p) + l.seq * t.seq + l.row * t.row + (l.sh - l.seq * heads) * t.head + c;
    return wide ? *reinterpret_cast<const float4*>(x) : make_float4(x[0], x[1], x[2], x[3]);
}

// blockIdx.y: the operand.  HD / 4 threads a line, ILP lines a thread.  Infinities and NaN
// do not count: they make their own products NaN whatever the scale.
template <int HD>
__global__ void __launch_bounds__(THREADS) attention_absmax_kernel(const __grid_constant__ SplitArgs a) {
    constexpr int TPL = HD / 4, LINES = THREADS / TPL;
    __shared__ float part[THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const Operand& p = a.op[blockIdx.y];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = threadIdx.x % TPL * 4;
    if (a.backward && blockIdx.y == 3)
        for (int i = blockIdx.x * THREADS + threadIdx.x; i < a.heads_total; i += gridDim.x * THREADS)
            a.sp.head_norm[i] = 0.0f;
    float m = 0.0f;
    for (long long first = (long long)blockIdx.x * LINES * ILP; first < p.lines; first += (long long)gridDim.x * LINES * ILP) {
        float4 v[ILP];
#pragma unroll
        for (int j = 0; j < ILP; j++) {
            v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const long long i = first + j * LINES + threadIdx.x / TPL;
            if (i < p.lines) {
                const Line l = line_of(p, (int)i);
                if (l.live) v[j] = line_load(p.t, l, p.heads, c, p.wide);
            }
        }
#pragma unroll
        for (int j = 0; j < ILP; j++) {
            const float x[4] = {fabsf(v[j].x), fabsf(v[j].y), fabsf(v[j].z), fabsf(v[j].w)};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (x[e] < INFINITY) m = fmaxf(m, x[e]);
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

template <int HD>
__global__ void __launch_bounds__(THREADS) attention_split_kernel(const __grid_constant__ SplitArgs a) {
    constexpr int TPL = HD / 4, LINES = THREADS / TPL;
    __shared__ float part[THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const Operand& p = a.op[blockIdx.y];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = threadIdx.x % TPL * 4;
    float m = 0.0f;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += THREADS) m = fmaxf(m, a.sp.partial[blockIdx.y * kSplitBlocks + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) part[warp] = m;
    __syncthreads();
    m = part[0];
    for (int i = 1; i < THREADS / 32; i++) m = fmaxf(m, part[i]);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.sp.maxima[blockIdx.y] = m;
    const float s = split_scale_of(m);
    const bool stats = a.backward && blockIdx.y == 3;
    // the largest |dout row| of the head that this thread is at: a maximum of non-negative floats, the same
    // in any order
    int norm_head = 0;
    float norm = 0.0f;
    auto keep_norm = [&](int next) {
        if (norm > 0.0f) atomicMax(reinterpret_cast<int*>(a.sp.head_norm + norm_head), __float_as_int(norm));
        norm_head = next;
        norm = 0.0f;
    };
    for (long long first = (long long)blockIdx.x * LINES * ILP; first < p.lines; first += (long long)gridDim.x * LINES * ILP) {
        float4 v[ILP], o[ILP];
        Line l[ILP];
        long long at[ILP];
#pragma unroll
        for (int j = 0; j < ILP; j++) {
            v[j] = o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            at[j] = first + j * LINES + threadIdx.x / TPL;
            l[j] = line_of(p, (int)min(at[j], (long long)p.lines - 1));
            if (l[j].live) {
                v[j] = line_load(p.t, l[j], p.heads, c, p.wide);
                if (stats) o[j] = line_load(a.o, l[j], p.heads, c, a.o_wide);
            }
        }
#pragma unroll
        for (int j = 0; j < ILP; j++) {
            const bool inside = at[j] < p.lines;
            uint2 h, lo;
            const float x[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            split2x4(x, s, h, lo);
            if (inside) {
                __half* out = p.out + at[j] * HD + c;
                *reinterpret_cast<uint2*>(out) = h;
                *reinterpret_cast<uint2*>(out + (long long)p.lines * HD) = lo;
            }
            if (stats) {
                float dot = x[0] * o[j].x + x[1] * o[j].y + x[2] * o[j].z + x[3] * o[j].w;
                float norm2 = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
                for (int k = TPL / 2; k > 0; k >>= 1) {
                    dot += __shfl_xor_sync(0xffffffffu, dot, k);
                    norm2 += __shfl_xor_sync(0xffffffffu, norm2, k);
                }
                if (inside && c == 0) {
                    const int row = l[j].row;
                    float* const tiles = a.sp.stats + (long long)l[j].sh * a.q_tiles * 2 * kSplitStat;
                    float* st = tiles + row / 64 * kSplitStat + row % 64;
                    const float lse = l[j].live ? a.lse[(long long)l[j].sh * p.rows + row] : -INFINITY;
                    st[0] = lse == -INFINITY ? -INFINITY : -lse * LOG2E;
                    st[64] = -dot;
                    st[128] = sqrtf(norm2);
                    if (l[j].sh != norm_head) keep_norm(l[j].sh);
                    if (norm2 > 0.0f) norm = fmaxf(norm, sqrtf(norm2));
                    // the rows of the last block of 64 that do not exist belong to it too
                    if (row == p.rows - 1)
                        for (int r = p.rows; r % 64 != 0; r++) {
                            float* e = tiles + r / 64 * kSplitStat + r % 64;
                            e[0] = -INFINITY;
                            e[64] = 0.0f;
                            e[128] = 0.0f;
                        }
                }
            }
        }
    }
    if (stats) keep_norm(0);
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
    auto wide = [](const HeadsView& v) {
        return reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && v.seq % 4 == 0 && v.row % 4 == 0 && v.head % 4 == 0;
    };
    long long most = 0;
    for (int i = 0; i < (backward ? 4 : 3); i++) {
        const bool keys = i == 1 || i == 2;
        Operand& p = t.op[i];
        p.t = views[i];
        p.len = keys ? a.k_len : a.q_len;
        p.rows = keys ? a.k_rows : a.q_rows;
        p.heads = keys ? a.k_heads : a.q_heads;
        const long long lines = (long long)a.seqs * p.heads * p.rows;
        if (lines > INT_MAX) throw Error(13, "attention: more than 2^31 rows of heads");
        p.lines = (int)lines;
        p.wide = wide(p.t);
        p.out = static_cast<__half*>(outs[i]);
        most = std::max(most, lines);
    }
    t.o = a.o;
    t.o_wide = wide(a.o);
    t.lse = a.lse;
    t.sp = sp;
    t.heads_total = a.seqs * a.q_heads;
    t.q_tiles = (a.q_rows + 127) / 128;
    t.backward = backward;
    const long long per = (long long)THREADS / (a.head_dim / 4) * ILP;
    const dim3 grid((unsigned)std::clamp<long long>((most + per - 1) / per, 1, kSplitBlocks), backward ? 4 : 3);
    if (a.head_dim == 64) {
        launch_pdl(attention_absmax_kernel<64>, grid, dim3(THREADS), 0, s, t);
        launch_pdl(attention_split_kernel<64>, grid, dim3(THREADS), 0, s, t);
    } else {
        launch_pdl(attention_absmax_kernel<128>, grid, dim3(THREADS), 0, s, t);
        launch_pdl(attention_split_kernel<128>, grid, dim3(THREADS), 0, s, t);
    }
}

}  // namespace n3d
