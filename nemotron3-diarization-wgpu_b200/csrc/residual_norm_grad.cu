// The gradient of r = x + scale * gate * Norm_post(block), y = Norm_pre(r)
// (n3d_residual_norm_grad).
//
// With h = (r - mean) / dev, g = dy * w_pre and means over the row (LayerNorm; RMS norm
// has no mean of r and no mean of g):
//   dx = dr + (g - mean g - h mean(g h)) / dev
//   dw_pre += dy h, db_pre += dy
// and with k = (block - mean) / dev, u = k w_post + b_post, e = scale * gate * dx * w_post:
//   dgate += scale dx u, dw_post += scale gate dx k, db_post += scale gate dx
//   dblock = (e - mean e - k mean(e k)) / dev
// Row statistics are taken again from r and block, which are read anyway: nothing of the
// forward call is kept, and the statistics are those of the r at hand.
//
// Bound: memory (r, dr, block, dy read once, dx, dblock written once).  The column sums
// (weights, biases, gate) stay in registers: a row's columns belong to the same threads
// for all rows of a slot, 8 columns a thread, so each of the five sums costs 8 registers.
// A slot is a contiguous range of rows; the next row's loads are issued before the
// current row's three sums over the row.  Slots of a block are added through shared
// memory, blocks by a second kernel, in a fixed order.  A gate row's gradient is complete
// when its rows lie in one slot; at the borders of slots partial sums go to the workspace
// and the second kernel adds them.

#include <algorithm>
#include <climits>

#include "residual_norm.cuh"

namespace n3d {

namespace {

constexpr int EPT = 8;  // columns of a thread

__host__ __device__ inline long long slot_begin(long long rows, int slots, int i) { return rows * i / slots; }

template <class RT, class BT, int VEC, int TPR>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, TPR > 256 ? 1 : 2)
    residual_norm_grad_kernel(const __grid_constant__ ResidualArgs a) {
    constexpr int CH = EPT / VEC;
    constexpr int THREADS = TPR > 256 ? TPR : 256, SLOTS = THREADS / TPR;
    __shared__ float sums[SLOTS][9][TPR / 32];
    __shared__ float part[SLOTS > 1 ? THREADS * EPT : 1];
    griddep_wait();
    griddep_launch_dependents();
    const int local = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const int slot = blockIdx.x * SLOTS + local;
    const int C = a.cols;
    const float inv_c = 1.0f / (float)C;
    float dgate[EPT] = {}, dpw[EPT] = {}, dpb[EPT] = {}, dqw[EPT] = {}, dqb[EPT] = {};  // p: post, q: pre
    const bool pre = a.pre != N3D_NORM_NONE, post = a.post != N3D_NORM_NONE;

    if (slot < a.slots) {
        const long long begin = slot_begin(a.rows, a.slots, slot), end = slot_begin(a.rows, a.slots, slot + 1);
        Vec<RT, VEC> rv[CH], drv[CH];
        Vec<BT, VEC> bv[CH], dyv[CH];
        auto fetch = [&](long long row) {
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                if (c < C) {
                    if (pre) {
                        rv[k].load_rw(static_cast<const RT*>(a.r) + row * a.ld_r + c);
                        dyv[k].load_rw(static_cast<const BT*>(a.dy) + row * a.ld_dy + c);
                    }
                    if (a.dr) drv[k].load_rw(static_cast<const RT*>(a.dr) + row * a.ld_dr + c);
                    bv[k].load_rw(static_cast<const BT*>(a.block) + row * a.ld_block + c);
                }
            }
        };
        // the gate row of the rows summed in dgate; flushed when it ends
        long long gate_row = a.rows_per_gate ? begin / a.rows_per_gate : 0;
        long long gate_end = a.rows_per_gate ? (gate_row + 1) * a.rows_per_gate : LLONG_MAX;
        auto flush_gate = [&](long long upto) {  // rows below `upto` are summed
            const long long g0 = gate_row * a.rows_per_gate, g1 = min(g0 + a.rows_per_gate, a.rows);
            float* out = a.dgate + gate_row * C;
            if (g0 < begin)
                out = a.gate_parts + (long long)slot * 2 * C;  // began in an earlier slot
            else if (g1 > upto)
                out = a.gate_parts + ((long long)slot * 2 + 1) * C;  // ends in a later one
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                if (c < C) {
                    if constexpr (VEC == 1) {
                        out[c] = dgate[k];
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; i += 4)
                            *reinterpret_cast<float4*>(out + c + i) =
                                make_float4(dgate[k * VEC + i], dgate[k * VEC + i + 1], dgate[k * VEC + i + 2],
                                            dgate[k * VEC + i + 3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < EPT; i++) dgate[i] = 0.0f;
        };

        fetch(begin);
        for (long long row = begin; row < end; row++) {
            float h[EPT], g[EPT], b[EPT], d[EPT];  // r (then h), dy (then g), block (then k), dr (then dx)
#pragma unroll
            for (int i = 0; i < EPT; i++) h[i] = g[i] = b[i] = d[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < CH; k++)
                if (chunk_col<VEC, TPR>(k, t) < C) {
                    if (pre) {
                        rv[k].get(h + k * VEC);
                        dyv[k].get(g + k * VEC);
                    }
                    if (a.dr) drv[k].get(d + k * VEC);
                    bv[k].get(b + k * VEC);
                }
            if (row + 1 < end) fetch(row + 1);
            if (a.rows_per_gate && row == gate_end) {
                if (a.dgate) flush_gate(row);
                gate_row++;
                gate_end += a.rows_per_gate;
            }
            float dy[EPT];
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                float w[VEC];
                if (pre && c < C) load_weights<VEC>(a.pre_w, c, 1.0f, w);
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    dy[k * VEC + i] = g[k * VEC + i];
                    if (pre && c < C) g[k * VEC + i] *= w[i];
                }
            }
            // ---- sums of r, block and g
            float s1[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < EPT; i++) s1[0] += h[i], s1[1] += b[i], s1[2] += g[i];
            row_sums<TPR>(s1, sums[local][0], local);
            const float mean_r = a.pre == N3D_NORM_LAYER ? s1[0] * inv_c : 0.0f;
            const float mean_b = a.post == N3D_NORM_LAYER ? s1[1] * inv_c : 0.0f;
            const float mean_g = a.pre == N3D_NORM_LAYER ? s1[2] * inv_c : 0.0f;
            // ---- squares of the centred values, and g against r
            float s2[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < CH; k++)
                if (chunk_col<VEC, TPR>(k, t) < C)
#pragma unroll
                    for (int i = k * VEC; i < (k + 1) * VEC; i++) {
                        h[i] -= mean_r;
                        b[i] -= mean_b;
                        s2[0] += h[i] * h[i];
                        s2[1] += b[i] * b[i];
                        s2[2] += g[i] * h[i];
                    }
            row_sums<TPR>(s2, sums[local][3], local);
            const float rstd_r = pre ? rsqrtf(s2[0] * inv_c + a.pre_eps) : 0.0f;
            const float rstd_b = post ? rsqrtf(s2[1] * inv_c + a.post_eps) : 1.0f;
            const float mean_gh = s2[2] * inv_c * rstd_r;
            const float* gate = a.rows_per_gate ? a.gate + gate_row * C : nullptr;
            float s3[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                if (c >= C) continue;
                float gt[VEC], w[VEC], bias[VEC];
                load_weights<VEC>(gate, c, 1.0f, gt);
                load_weights<VEC>(post ? a.post_w : nullptr, c, 1.0f, w);
                load_weights<VEC>(post ? a.post_b : nullptr, c, 0.0f, bias);
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const int i = k * VEC + j;
                    h[i] *= rstd_r;
                    d[i] += rstd_r * (g[i] - mean_g - h[i] * mean_gh);
                    dqw[i] += dy[i] * h[i];
                    dqb[i] += dy[i];
                    b[i] *= rstd_b;
                    const float sd = a.scale * d[i];
                    dgate[i] += sd * (b[i] * w[j] + bias[j]);
                    const float du = sd * gt[j];
                    dpw[i] += du * b[i];
                    dpb[i] += du;
                    g[i] = du * w[j];  // e
                    s3[0] += g[i];
                    s3[1] += g[i] * b[i];
                }
                Vec<RT, VEC> o;
                o.set(d + k * VEC);
                o.store(static_cast<RT*>(a.dx) + row * a.ld_dx + c);
            }
            // ---- e, and e against k
            float mean_e = 0.0f, mean_ek = 0.0f;
            if (post) {
                row_sums<TPR>(s3, sums[local][6], local);
                mean_e = a.post == N3D_NORM_LAYER ? s3[0] * inv_c : 0.0f;
                mean_ek = s3[1] * inv_c;
            }
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                if (c >= C) continue;
#pragma unroll
                for (int i = k * VEC; i < (k + 1) * VEC; i++) g[i] = rstd_b * (g[i] - mean_e - b[i] * mean_ek);
                Vec<BT, VEC> o;
                o.set(g + k * VEC);
                o.store(static_cast<BT*>(a.dblock) + row * a.ld_dblock + c);
            }
        }
        if (a.dgate) flush_gate(end);
    }
    // ---- the block's slots, then its sums to the workspace
    float* mine = a.sums + (long long)blockIdx.x * 4 * C;
    auto emit = [&](float (&v)[EPT], int which) {
        if constexpr (SLOTS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < EPT; i++) part[(local * EPT + i) * TPR + t] = v[i];
            __syncthreads();
            if (local == 0)
#pragma unroll
                for (int i = 0; i < EPT; i++)
                    for (int o = 1; o < SLOTS; o++) v[i] += part[(o * EPT + i) * TPR + t];
        }
        if (local == 0)
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                if (c < C)
#pragma unroll
                    for (int i = 0; i < VEC; i++) mine[(long long)which * C + c + i] = v[k * VEC + i];
            }
    };
    if (a.dpost_w) emit(dpw, 0);
    if (a.dpost_b) emit(dpb, 1);
    if (a.dpre_w) emit(dqw, 2);
    if (a.dpre_b) emit(dqb, 3);
}

// Adds the partial sums: blockIdx.y < 4 the blocks' weight and bias sums, the others the
// gate rows that lie in several slots.  These are looked for among the `items` gate rows
// (by_row), or where there are fewer borders between slots than gate rows, among the rows
// at the borders.  8 threads per column, joined in a fixed order.
__global__ void __launch_bounds__(256)
    residual_norm_finish_kernel(const __grid_constant__ ResidualArgs a, int blocks, long long items, int by_row) {
    __shared__ float part[8][32];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const long long C = a.cols;
    auto add = [&](const float* first, const float* later, long long step, int n, float* dst) {
        float v = 0.0f;
        if (c < C)
#pragma unroll 4
            for (int k = w; k < n; k += 8) v += k == 0 ? first[c] : later[k * step + c];
        part[w][lane] = v;
        __syncthreads();
        if (w == 0 && c < C) {
#pragma unroll
            for (int k = 1; k < 8; k++) v += part[k][lane];
            dst[c] = v;
        }
        __syncthreads();
    };
    if (blockIdx.y < 4) {
        float* const dst = blockIdx.y == 0 ? a.dpost_w : blockIdx.y == 1 ? a.dpost_b : blockIdx.y == 2 ? a.dpre_w : a.dpre_b;
        const float* src = a.sums + blockIdx.y * C;
        if (dst) add(src, src, 4 * C, blocks, dst);
        return;
    }
    auto slot_of = [&](long long row) { return (int)(((row + 1) * a.slots - 1) / a.rows); };
    for (long long i = blockIdx.y - 4; i < items; i += gridDim.y - 4) {
        const long long g = by_row ? i : slot_begin(a.rows, a.slots, (int)i + 1) / a.rows_per_gate;
        const long long g0 = g * a.rows_per_gate, g1 = min(g0 + a.rows_per_gate, a.rows);
        const int s0 = slot_of(g0), s1 = slot_of(g1 - 1);
        // in one slot: complete already; several borders inside one gate row: done by the first
        if (s0 == s1 || (!by_row && s0 != i)) continue;
        const float* parts = a.gate_parts + (long long)s0 * 2 * C;
        add(parts + C, parts, 2 * C, s1 - s0 + 1, a.dgate + g * C);
    }
}

template <class RT, class BT, int VEC, int TPR>
void launch(cudaStream_t s, const ResidualArgs& a, const ResidualSplit& sp) {
    constexpr int THREADS = TPR > 256 ? TPR : 256;
    launch_pdl(residual_norm_grad_kernel<RT, BT, VEC, TPR>, dim3(sp.blocks), dim3(THREADS), 0, s, a);
}

template <class RT, class BT>
void launch_type(cudaStream_t s, const ResidualArgs& a, const ResidualSplit& sp) {
    if (!a.wide) {
        sp.threads == 128 ? launch<RT, BT, 1, 128>(s, a, sp) : launch<RT, BT, 1, 1024>(s, a, sp);
        return;
    }
    switch (sp.threads) {
        case 32: return launch<RT, BT, 8, 32>(s, a, sp);
        case 64: return launch<RT, BT, 8, 64>(s, a, sp);
        case 128: return launch<RT, BT, 8, 128>(s, a, sp);
        case 256: return launch<RT, BT, 8, 256>(s, a, sp);
        case 512: return launch<RT, BT, 8, 512>(s, a, sp);
        default: return launch<RT, BT, 8, 1024>(s, a, sp);
    }
}

}  // namespace

// Two blocks of 256 threads fit an SM, one of 512 or 1024: 148 SMs' worth of blocks, and
// no more slots than rows.  (The count is fixed, so that results do not depend on the GPU.)
ResidualSplit residual_split(long long rows, int cols, bool wide) {
    ResidualSplit sp;
    if (wide) {
        sp.threads = 32;
        while (sp.threads * EPT < cols) sp.threads *= 2;
    } else {
        sp.threads = cols <= 128 * EPT ? 128 : 1024;
    }
    const int block = std::max(sp.threads, 256);
    sp.per_block = block / sp.threads;
    const long long most = (block == 256 ? 296LL : 148LL) * sp.per_block;
    sp.slots = (int)std::max<long long>(1, std::min(most, rows));
    sp.blocks = (sp.slots + sp.per_block - 1) / sp.per_block;
    return sp;
}

void launch_residual_norm_grad(cudaStream_t s, const ResidualArgs& a, int residual_dtype, int block_dtype) {
    const ResidualSplit sp = residual_split(a.rows, a.cols, a.wide);
    if (residual_dtype == N3D_BF16)
        launch_type<__nv_bfloat16, __nv_bfloat16>(s, a, sp);
    else if (residual_dtype == N3D_F16)
        launch_type<__half, __half>(s, a, sp);
    else if (block_dtype == N3D_BF16)
        launch_type<float, __nv_bfloat16>(s, a, sp);
    else if (block_dtype == N3D_F16)
        launch_type<float, __half>(s, a, sp);
    else
        launch_type<float, float>(s, a, sp);
    const bool weights = a.dpost_w || a.dpost_b || a.dpre_w || a.dpre_b;
    const long long gates = a.dgate ? (a.rows + a.rows_per_gate - 1) / a.rows_per_gate : 0;
    const long long items = a.dgate && sp.slots > 1 ? std::min<long long>(gates, sp.slots - 1) : 0;
    if (weights || items > 0)
        launch_pdl(residual_norm_finish_kernel, dim3((a.cols + 31) / 32, 4 + (unsigned)std::min<long long>(items, 32)),
                   dim3(256), 0, s, a, sp.blocks, items, (int)(gates <= items));
}

}  // namespace n3d
