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
// Bound: memory (r, dr, block, dy read once, dx, dblock written once); what costs time is
// the latency of two or three sums over each row, so that many rows must be in work.  A row
// has one thread for every 8 columns (16 beyond 4096), and a slot of threads takes a
// contiguous range of rows, two at a time (one beyond 4096): their sums share the barriers, and the weights
// are read and the column sums (weights, biases, gate; in shared memory, where each thread
// alone adds to its columns) updated once for both.  One row at a time with the column sums
// in registers, up to 40 a thread, took 176 us for 8191 x 4096 in bf16; two take 124.  Slots of
// a block are added at the end, blocks by a second kernel, in a fixed order.  A gate row's
// gradient is complete when its rows lie in one slot; at the borders of slots partial sums
// go to the workspace and the second kernel adds them.
//
// Measured on a B200: 48128 x 512, fp32 stream and bf16 blocks, LayerNorms and a gate 111 us
// (4.0 TB/s); fp32 throughout without a gate 104 us (5.7 TB/s); 8191 x 4096 in bf16, RMS norms
// and gates 124 us (3.2 TB/s; the registers of 512 threads, one pair of rows, fill an SM).

#include <algorithm>
#include <climits>

#include "residual_norm.cuh"

namespace n3d {

namespace {

__host__ __device__ inline long long slot_begin(long long rows, int slots, int i) { return rows * i / slots; }

// TPR threads a row, EPT columns a thread, R rows at a time.
template <int TPR, int EPT>
struct GradCfg {
    static constexpr int THREADS = TPR > 256 ? TPR : 256, SLOTS = THREADS / TPR, PER_SM = 512 / THREADS;
    static constexpr int SUM = THREADS * EPT;  // floats of one column sum of the block
    static constexpr int BYTES = 5 * SUM * 4;
};
enum { POST_W, POST_B, PRE_W, PRE_B, GATE };  // the column sums

template <class RT, class BT, int VEC, int TPR, int EPT, int R>
__global__ void __launch_bounds__(GradCfg<TPR, EPT>::THREADS, GradCfg<TPR, EPT>::PER_SM)
    residual_norm_grad_kernel(const __grid_constant__ ResidualArgs a) {
    using Cfg = GradCfg<TPR, EPT>;
    constexpr int CH = EPT / VEC, SLOTS = Cfg::SLOTS;
    extern __shared__ float4 smem4[];
    __shared__ float sums[SLOTS][8 * R][TPR / 32];
    griddep_wait();
    griddep_launch_dependents();
    const int local = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const int slot = blockIdx.x * SLOTS + local;
    const int C = a.cols;
    const float inv_c = 1.0f / (float)C;
    const bool pre = a.pre != N3D_NORM_NONE, post = a.post != N3D_NORM_NONE;
    // this thread's values of a column sum: 16-byte words, those of neighbours side by side
    float* const mine = reinterpret_cast<float*>(smem4) + 4 * threadIdx.x;
    auto at = [&](int which, int i) -> float4& {  // its columns 4 i ..
        return *reinterpret_cast<float4*>(mine + which * Cfg::SUM + i * (Cfg::THREADS * 4));
    };
    auto add = [&](int which, int k, const float (&v)[VEC]) {  // the columns of chunk k
        if constexpr (VEC == 4) {
            float4 f = at(which, k);
            f.x += v[0], f.y += v[1], f.z += v[2], f.w += v[3];
            at(which, k) = f;
        } else {
            (&at(which, k / 4).x)[k % 4] += v[0];
        }
    };
#pragma unroll
    for (int k = 0; k < 5; k++)
#pragma unroll
        for (int i = 0; i < EPT / 4; i++) at(k, i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

    if (slot < a.slots) {
        const long long begin = slot_begin(a.rows, a.slots, slot), end = slot_begin(a.rows, a.slots, slot + 1);
        // the gate row of the rows summed so far; flushed when it ends
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
            for (int i = 0; i < EPT / 4; i++) {
                const float4 f = at(GATE, i);
                at(GATE, i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if constexpr (VEC == 1) {
                    const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (chunk_col<1, TPR>(4 * i + j, t) < C) out[chunk_col<1, TPR>(4 * i + j, t)] = v[j];
                } else if (chunk_col<VEC, TPR>(i, t) < C) {
                    *reinterpret_cast<float4*>(out + chunk_col<VEC, TPR>(i, t)) = f;
                }
            }
        };

        // With an RMS norm (or none) before and none behind, only the second sum below is taken.  A sum's words may be
        // written again only past another barrier of the row, so that sum then takes its own words and those of
        // the first one in turn.
        const bool alone = a.pre != N3D_NORM_LAYER && !post;
        bool turn = false;
        long long row = begin;
        while (row < end) {
            if (row == gate_end) {
                if (a.dgate) flush_gate(row);
                gate_row++;
                gate_end += a.rows_per_gate;
            }
            // R rows of one gate row, or what is left of it; the others are zeros, which add nothing
            const int n = (int)min((long long)R, min(end, gate_end) - row);
            Vec<RT, VEC> drv[R][CH];
            Vec<BT, VEC> dyv[R][CH];
            float h[R][EPT], g[R][EPT], b[R][EPT];  // r (then h), dy w (then e), block (then k)
            {
                Vec<RT, VEC> rv[R][CH];
                Vec<BT, VEC> bv[R][CH];
#pragma unroll
                for (int q = 0; q < R; q++)
#pragma unroll
                    for (int k = 0; k < CH; k++) {
                        const int c = chunk_col<VEC, TPR>(k, t);
                        rv[q][k] = {}, dyv[q][k] = {}, bv[q][k] = {}, drv[q][k] = {};
                        if (c < C && q < n) {
                            if (pre) {
                                rv[q][k].load_rw(static_cast<const RT*>(a.r) + (row + q) * a.ld_r + c);
                                dyv[q][k].load_rw(static_cast<const BT*>(a.dy) + (row + q) * a.ld_dy + c);
                            }
                            bv[q][k].load_rw(static_cast<const BT*>(a.block) + (row + q) * a.ld_block + c);
                            if (a.dr) drv[q][k].load_rw(static_cast<const RT*>(a.dr) + (row + q) * a.ld_dr + c);
                        }
                    }
#pragma unroll
                for (int k = 0; k < CH; k++) {
                    const int c = chunk_col<VEC, TPR>(k, t);
                    float w[VEC];
                    load_weights<VEC>(c < C ? a.pre_w : nullptr, c, 1.0f, w);
#pragma unroll
                    for (int q = 0; q < R; q++) {
                        rv[q][k].get(h[q] + k * VEC);
                        dyv[q][k].get(g[q] + k * VEC);
                        bv[q][k].get(b[q] + k * VEC);
#pragma unroll
                        for (int i = 0; i < VEC; i++) g[q][k * VEC + i] *= w[i];
                    }
                }
            }
            // ---- means of r, block and g, where a norm subtracts them
            float mean_g[R] = {};
            if (a.pre == N3D_NORM_LAYER || a.post == N3D_NORM_LAYER) {
                float s1[3 * R] = {};
#pragma unroll
                for (int q = 0; q < R; q++)
#pragma unroll
                    for (int i = 0; i < EPT; i++)
                        s1[3 * q] += h[q][i], s1[3 * q + 1] += b[q][i], s1[3 * q + 2] += g[q][i];
                row_sums<TPR>(s1, sums[local][0], local);
#pragma unroll
                for (int q = 0; q < R; q++) {
                    const float mean_r = a.pre == N3D_NORM_LAYER ? s1[3 * q] * inv_c : 0.0f;
                    const float mean_b = a.post == N3D_NORM_LAYER ? s1[3 * q + 1] * inv_c : 0.0f;
                    mean_g[q] = a.pre == N3D_NORM_LAYER ? s1[3 * q + 2] * inv_c : 0.0f;
#pragma unroll
                    for (int i = 0; i < EPT; i++) h[q][i] -= mean_r, b[q][i] -= mean_b;
                }
            }
            // ---- squares of the centred values, and g against r
            float s2[3 * R] = {};
#pragma unroll
            for (int k = 0; k < CH; k++)
                if (chunk_col<VEC, TPR>(k, t) < C)
#pragma unroll
                    for (int q = 0; q < R; q++)
#pragma unroll
                        for (int i = k * VEC; i < (k + 1) * VEC; i++) {
                            s2[3 * q] += h[q][i] * h[q][i];
                            s2[3 * q + 1] += b[q][i] * b[q][i];
                            s2[3 * q + 2] += g[q][i] * h[q][i];
                        }
            row_sums<TPR>(s2, sums[local][turn ? 0 : 3 * R], local);
            turn = alone && !turn;
            float rstd_b[R], s3[2 * R] = {};
            const float* gate = a.rows_per_gate ? a.gate + gate_row * C : nullptr;
#pragma unroll
            for (int q = 0; q < R; q++) {
                const float rstd_r = pre ? rsqrtf(s2[3 * q] * inv_c + a.pre_eps) : 0.0f;
                const float mean_gh = s2[3 * q + 2] * inv_c * rstd_r;
                rstd_b[q] = post ? rsqrtf(s2[3 * q + 1] * inv_c + a.post_eps) : 1.0f;
#pragma unroll
                for (int i = 0; i < EPT; i++) {
                    h[q][i] *= rstd_r;
                    g[q][i] = rstd_r * (g[q][i] - mean_g[q] - h[q][i] * mean_gh);
                    b[q][i] *= rstd_b[q];
                }
            }
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int c = chunk_col<VEC, TPR>(k, t);
                if (c >= C) continue;
                float v[VEC], d[VEC];
                // dy h and dy
                if (a.dpre_w || a.dpre_b) {
                    float u[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i++) u[i] = v[i] = 0.0f;
#pragma unroll
                    for (int q = 0; q < R; q++) {
                        dyv[q][k].get(d);
#pragma unroll
                        for (int i = 0; i < VEC; i++) u[i] += d[i], v[i] += d[i] * h[q][k * VEC + i];
                    }
                    if (a.dpre_w) add(PRE_W, k, v);
                    if (a.dpre_b) add(PRE_B, k, u);
                }
                // dx; from here g is scale dx
#pragma unroll
                for (int q = 0; q < R; q++) {
                    float* gq = g[q] + k * VEC;
                    if (a.dr) {
                        drv[q][k].get(d);
#pragma unroll
                        for (int i = 0; i < VEC; i++) gq[i] += d[i];
                    }
                    if (q < n) {
                        Vec<RT, VEC> o;
                        o.set(gq);
                        o.store(static_cast<RT*>(a.dx) + (row + q) * a.ld_dx + c);
                    }
#pragma unroll
                    for (int i = 0; i < VEC; i++) gq[i] *= a.scale;
                }
                float w[VEC];
                load_weights<VEC>(post ? a.post_w : nullptr, c, 1.0f, w);
                if (a.dgate) {
                    load_weights<VEC>(post ? a.post_b : nullptr, c, 0.0f, d);
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        v[i] = 0.0f;
#pragma unroll
                        for (int q = 0; q < R; q++) v[i] += g[q][k * VEC + i] * (b[q][k * VEC + i] * w[i] + d[i]);
                    }
                    add(GATE, k, v);
                }
                load_weights<VEC>(gate, c, 1.0f, d);
#pragma unroll
                for (int q = 0; q < R; q++)
#pragma unroll
                    for (int i = 0; i < VEC; i++) g[q][k * VEC + i] *= d[i];
                if (a.dpost_b) {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        v[i] = 0.0f;
#pragma unroll
                        for (int q = 0; q < R; q++) v[i] += g[q][k * VEC + i];
                    }
                    add(POST_B, k, v);
                }
                if (a.dpost_w) {
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        v[i] = 0.0f;
#pragma unroll
                        for (int q = 0; q < R; q++) v[i] += g[q][k * VEC + i] * b[q][k * VEC + i];
                    }
                    add(POST_W, k, v);
                }
                // e, and e against k
#pragma unroll
                for (int q = 0; q < R; q++)
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        float& e = g[q][k * VEC + i];
                        e *= w[i];
                        s3[2 * q] += e;
                        s3[2 * q + 1] += e * b[q][k * VEC + i];
                    }
            }
            if (post) row_sums<TPR>(s3, sums[local][6 * R], local);
#pragma unroll
            for (int q = 0; q < R; q++) {
                if (q >= n) continue;
                const float mean_e = a.post == N3D_NORM_LAYER ? s3[2 * q] * inv_c : 0.0f;
                const float mean_ek = post ? s3[2 * q + 1] * inv_c : 0.0f;
#pragma unroll
                for (int k = 0; k < CH; k++) {
                    const int c = chunk_col<VEC, TPR>(k, t);
                    if (c >= C) continue;
                    float v[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        v[i] = rstd_b[q] * (g[q][k * VEC + i] - mean_e - b[q][k * VEC + i] * mean_ek);
                    Vec<BT, VEC> o;
                    o.set(v);
                    o.store(static_cast<BT*>(a.dblock) + (row + q) * a.ld_dblock + c);
                }
            }
            row += n;
        }
        if (a.dgate) flush_gate(end);
    }
    // ---- the slots of the block in order, to the workspace
    __syncthreads();
    float* out = a.sums + (long long)blockIdx.x * 4 * C;
    for (int which = 0; which < 4; which++) {
        const float* wanted = which == POST_W ? a.dpost_w : which == POST_B ? a.dpost_b : which == PRE_W ? a.dpre_w : a.dpre_b;
        if (!wanted || local != 0) continue;
#pragma unroll
        for (int i = 0; i < EPT / 4; i++) {
            float4 f = at(which, i);
            for (int o = 1; o < SLOTS; o++) {
                const float4 e = *(&at(which, i) + o * TPR);
                f.x += e.x, f.y += e.y, f.z += e.z, f.w += e.w;
            }
            const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int c = VEC == 1 ? chunk_col<VEC, TPR>(4 * i + j, t) : chunk_col<VEC, TPR>(i, t) + j;
                if (c < C) out[(long long)which * C + c] = v[j];
            }
        }
    }
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

template <class RT, class BT, int VEC, int TPR, int EPT, int R>
void launch(cudaStream_t s, const ResidualArgs& a, const ResidualSplit& sp) {
    using Cfg = GradCfg<TPR, EPT>;
    static std::atomic<unsigned long long> attr{0};
    once_per_device(attr, [] {
        N3D_CUDA(cudaFuncSetAttribute(residual_norm_grad_kernel<RT, BT, VEC, TPR, EPT, R>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::BYTES));
    });
    launch_pdl(residual_norm_grad_kernel<RT, BT, VEC, TPR, EPT, R>, dim3(sp.blocks), dim3(Cfg::THREADS), Cfg::BYTES, s, a);
}

template <class RT, class BT>
void launch_type(cudaStream_t s, const ResidualArgs& a, const ResidualSplit& sp) {
    if (!a.wide) {
        sp.threads == 128 ? launch<RT, BT, 1, 128, 8, 2>(s, a, sp) : launch<RT, BT, 1, 512, 16, 1>(s, a, sp);
        return;
    }
    switch (sp.threads * (a.cols > 4096 ? 2 : 1)) {
        case 32: return launch<RT, BT, 4, 32, 8, 2>(s, a, sp);
        case 64: return launch<RT, BT, 4, 64, 8, 2>(s, a, sp);
        case 128: return launch<RT, BT, 4, 128, 8, 2>(s, a, sp);
        case 256: return launch<RT, BT, 4, 256, 8, 2>(s, a, sp);
        case 512: return launch<RT, BT, 4, 512, 8, 2>(s, a, sp);
        default: return launch<RT, BT, 4, 512, 16, 1>(s, a, sp);
    }
}

}  // namespace

// 512 threads fit an SM (128 registers each): 148 SMs' worth of blocks, and no more slots
// than rows.  (The count is fixed, so that results do not depend on the GPU.)
ResidualSplit residual_split(long long rows, int cols, bool wide) {
    ResidualSplit sp;
    if (wide) {  // 8 columns a thread, 16 beyond 512 threads
        sp.threads = 32;
        while (sp.threads < 512 && sp.threads * 8 < cols) sp.threads *= 2;
    } else {
        sp.threads = cols <= 1024 ? 128 : 512;
    }
    const int block = std::max(sp.threads, 256);
    sp.per_block = block / sp.threads;
    const long long most = 148LL * (512 / block) * sp.per_block;
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
