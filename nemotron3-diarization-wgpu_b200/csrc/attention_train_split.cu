// fp32 operands of the training attention for the tensor cores: each row of q, k, v (and dout) as
// two fp16 arrays of x s (h = x s rounded to 11 bits, l the rest), as the library's other fp32
// products (n3d_device.cuh), with a power of two s for every row: the one that brings its largest
// magnitude into [2^14, 2^15).  The main kernel takes the rows' units 1 / s where it has a row or
// a column of scores in hand.  (One s for a whole tensor would leave a row 2^-20 the size of the
// largest with 20 bits, one of 2^-40 with none, and let a sequence's result depend on what else is in
// the batch.)  Rows past the lengths become zeros.
//
// For the gradient the same pass takes, per query row, -lse log2 e and -D = -(dout . out), in
// fp32 from the unsplit tensors.
//
// Bound: latency (four lines of a thread are in flight) before memory: one read of each
// operand and one write of the same size.  Measured on a B200, cold: q, k and v of 8 x 501 rows,
// 8 heads of 64 (25 MB) 18 - 20 us, with dout and the statistics 24 - 26; of 2 x 4096 rows, 16 heads (101 MB) 60 and 88.

#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "n3d_device.cuh"
#include "train.h"

namespace n3d {

namespace {

constexpr int THREADS = 256;
constexpr int ILP = 4;       // lines of a thread in flight
constexpr int BLOCKS = 296;  // at most, of each operand
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
    int q_tiles, k_tiles;  // blocks of 128 query rows, of 64 key rows
    int backward;
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

// The power of two that brings m into [2^14, 2^15), at most 2^126 so that its inverse is normal too; 1 for m = 0.
__device__ __forceinline__ float row_scale(float m) {
    if (!(m > 0.0f)) return 1.0f;
    return __int_as_float(min(253, 268 - (__float_as_int(m) >> 23)) << 23);
}

// blockIdx.y: the operand.  HD / 4 threads a line, ILP lines a thread.
template <int HD>
__global__ void __launch_bounds__(THREADS) attention_split_kernel(const __grid_constant__ SplitArgs a) {
    constexpr int TPL = HD / 4, LINES = THREADS / TPL;
    griddep_wait();
    griddep_launch_dependents();
    const int which = blockIdx.y;
    const Operand& p = a.op[which];
    const bool keys = which == 1 || which == 2, stats = a.backward && which == 3;
    const int c = threadIdx.x % TPL * 4;
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
            const float x[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            // the row's largest magnitude; infinities and NaN do not count: their products are NaN whatever the scale
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (fabsf(x[e]) < INFINITY) m = fmaxf(m, fabsf(x[e]));
            float dot = x[0] * o[j].x + x[1] * o[j].y + x[2] * o[j].z + x[3] * o[j].w;
#pragma unroll
            for (int k = TPL / 2; k > 0; k >>= 1) {
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
                if (stats) dot += __shfl_xor_sync(0xffffffffu, dot, k);
            }
            const float s = row_scale(m);
            if (!inside) continue;
            uint2 h, lo;
            split2x4(x, s, h, lo);
            __half* out = p.out + at[j] * HD + c;
            *reinterpret_cast<uint2*>(out) = h;
            *reinterpret_cast<uint2*>(out + (long long)p.lines * HD) = lo;
            if (c != 0) continue;
            // what the row's block of 64 holds of it; the rows of the last block that do not exist belong to the last row
            const int row = l[j].row, end = row == p.rows - 1 ? (row / 64 + 1) * 64 : row + 1;
            float* const blocks = keys ? a.sp.key_stats + (long long)l[j].sh * a.k_tiles * kKeyStat
                                       : a.sp.stats + (long long)l[j].sh * a.q_tiles * 2 * kSplitStat;
            float* const st = blocks + row / 64 * (keys ? kKeyStat : kSplitStat) + row % 64;
            const int unit = keys ? (which - 1) * 64 : which == 0 ? 128 : 192;
            for (int r = 0; r < end - row; r++) st[unit + r] = r == 0 ? 1.0f / s : 1.0f;
            if (stats) {
                const float lse = l[j].live ? a.lse[(long long)l[j].sh * p.rows + row] : -INFINITY;
                for (int r = 0; r < end - row; r++) {
                    st[r] = r > 0 || lse == -INFINITY ? -INFINITY : -lse * LOG2E;
                    st[64 + r] = r > 0 ? 0.0f : -dot;
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
    s.q = take(q);
    s.k = take(k);
    s.v = take(k);
    s.stats = static_cast<float*>(take(seqs * q_heads * ((q_rows + 127) / 128) * 2 * kSplitStat * sizeof(float)));
    s.key_stats = static_cast<float*>(take(seqs * k_heads * ((k_rows + 63) / 64) * kKeyStat * sizeof(float)));
    if (backward) s.dout = take(q);
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
    t.q_tiles = (a.q_rows + 127) / 128;
    t.k_tiles = (a.k_rows + 63) / 64;
    t.backward = backward;
    const long long per = (long long)THREADS / (a.head_dim / 4) * ILP;
    const dim3 grid((unsigned)std::clamp<long long>((most + per - 1) / per, 1, BLOCKS), backward ? 4 : 3);
    launch_pdl(a.head_dim == 64 ? attention_split_kernel<64> : attention_split_kernel<128>, grid, dim3(THREADS), 0, s, t);
}

}  // namespace n3d
