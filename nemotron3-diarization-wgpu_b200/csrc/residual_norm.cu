// r = x + scale * gate * Norm_post(block), y = Norm_pre(r) (n3d_residual_norm).
//
// Bound: memory.  Each element of x and block is read once and each of r and y written
// once; the row stays in registers between its sums (mean, then the squares of the
// centred values, for each norm), so nothing is read twice.  Rows of up to 1024 columns
// belong to one warp, whose sums need no barrier; wider rows to a block of 128 or 256
// threads with 16 or 32 columns each.  Enough warps are resident to keep loads in flight while
// others sum.
//
// Measured on a B200: 48128 x 512, fp32 stream and bf16 blocks, both norms and a gate, 48 us
// (6.1 TB/s); 8191 x 4096 the same 70 us (5.8 TB/s); in bf16 throughout, RMS norms, 66 us
// (4.0 TB/s); 4000 x 8192 the same 54 us (4.9 TB/s).

#include <algorithm>
#include <climits>

#include "residual_norm.cuh"

namespace n3d {

namespace {

template <class RT, class BT, int VEC, int TPR, int EPT>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128)
    residual_norm_kernel(const __grid_constant__ ResidualArgs a) {
    constexpr int CH = EPT / VEC;  // chunks of a thread
    constexpr int THREADS = TPR > 128 ? TPR : 128, SLOTS = THREADS / TPR;
    __shared__ float sums[SLOTS][4][TPR / 32];
    griddep_wait();
    griddep_launch_dependents();
    const int slot = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * SLOTS + slot;
    if (row >= a.rows) return;  // all threads of the row
    const int C = a.cols;
    const float inv_c = 1.0f / (float)C;
    const RT* x = static_cast<const RT*>(a.x) + row * a.ld_x;
    const BT* blk = static_cast<const BT*>(a.block) + row * a.ld_block;
    Vec<RT, VEC> xv[CH];
    Vec<BT, VEC> bv[CH];
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const int c = chunk_col<VEC, TPR>(k, t);
        if (c < C) {
            bv[k].load_rw(blk + c);
            xv[k].load_rw(x + c);
        }
    }
    float u[EPT];
#pragma unroll
    for (int k = 0; k < CH; k++) {
        if (chunk_col<VEC, TPR>(k, t) < C) {
            bv[k].get(u + k * VEC);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) u[k * VEC + i] = 0.0f;
        }
    }
    // centred values and 1 / deviation of v; columns past C stay 0
    auto normalise = [&](float (&v)[EPT], int kind, float eps, float* buf) {
        float s[1] = {0.0f}, mean = 0.0f;
        if (kind == N3D_NORM_LAYER) {
#pragma unroll
            for (int i = 0; i < EPT; i++) s[0] += v[i];
            row_sums<TPR>(s, buf, slot);
            mean = s[0] * inv_c;
        }
        s[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; k++)
            if (chunk_col<VEC, TPR>(k, t) < C)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    v[k * VEC + i] -= mean;
                    s[0] += v[k * VEC + i] * v[k * VEC + i];
                }
        row_sums<TPR>(s, buf + TPR / 32, slot);
        return rsqrtf(s[0] * inv_c + eps);
    };
    float rstd = 1.0f;
    if (a.post != N3D_NORM_NONE) rstd = normalise(u, a.post, a.post_eps, sums[slot][0]);
    const float* gate = a.rows_per_gate ? a.gate + row / a.rows_per_gate * C : nullptr;
    RT* r_out = static_cast<RT*>(a.r_out) + row * a.ld_r_out;
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const int c = chunk_col<VEC, TPR>(k, t);
        if (c < C) {
            float w[VEC], b[VEC], g[VEC], f[VEC];
            xv[k].get(f);
            load_weights<VEC>(gate, c, 1.0f, g);
            if (a.post != N3D_NORM_NONE) {
                load_weights<VEC>(a.post_w, c, 1.0f, w);
                load_weights<VEC>(a.post_b, c, 0.0f, b);
#pragma unroll
                for (int i = 0; i < VEC; i++) u[k * VEC + i] = u[k * VEC + i] * rstd * w[i] + b[i];
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) u[k * VEC + i] = f[i] + a.scale * (g[i] * u[k * VEC + i]);
            xv[k].set(u + k * VEC);
            xv[k].store(r_out + c);
        }
    }
    if (a.pre == N3D_NORM_NONE) return;
    rstd = normalise(u, a.pre, a.pre_eps, sums[slot][2]);
    BT* y = static_cast<BT*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int k = 0; k < CH; k++) {
        const int c = chunk_col<VEC, TPR>(k, t);
        if (c < C) {
            float w[VEC], b[VEC];
            load_weights<VEC>(a.pre_w, c, 1.0f, w);
            load_weights<VEC>(a.pre_b, c, 0.0f, b);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[k * VEC + i] = u[k * VEC + i] * rstd * w[i] + b[i];
            bv[k].set(u + k * VEC);
            bv[k].store(y + c);
        }
    }
}

template <class RT, class BT, int VEC, int TPR, int EPT>
void launch(cudaStream_t s, const ResidualArgs& a) {
    constexpr int THREADS = TPR > 128 ? TPR : 128, SLOTS = THREADS / TPR;
    const long long blocks = (a.rows + SLOTS - 1) / SLOTS;
    if (blocks > INT_MAX) throw Error(13, "n3d_residual_norm: more than 2^31 blocks of rows");
    launch_pdl(residual_norm_kernel<RT, BT, VEC, TPR, EPT>, dim3((unsigned)blocks), dim3(THREADS), 0, s, a);
}

template <class RT, class BT>
void launch_type(cudaStream_t s, const ResidualArgs& a) {
    const int C = a.cols;
    if (!a.wide)
        C <= 1024 ? launch<RT, BT, 1, 32, 32>(s, a) : launch<RT, BT, 1, 256, 32>(s, a);
    else if (C <= 256)
        launch<RT, BT, 4, 32, 8>(s, a);
    else if (C <= 512)
        launch<RT, BT, 4, 32, 16>(s, a);
    else if (C <= 1024)
        launch<RT, BT, 4, 32, 32>(s, a);
    else if (C <= 2048)
        launch<RT, BT, 4, 128, 16>(s, a);
    else if (C <= 4096)
        launch<RT, BT, 4, 256, 16>(s, a);
    else
        launch<RT, BT, 4, 256, 32>(s, a);
}

}  // namespace

void launch_residual_norm(cudaStream_t s, const ResidualArgs& a, int residual_dtype, int block_dtype) {
    if (a.rows <= 0) return;
    if (residual_dtype == N3D_BF16)
        launch_type<__nv_bfloat16, __nv_bfloat16>(s, a);
    else if (residual_dtype == N3D_F16)
        launch_type<__half, __half>(s, a);
    else if (block_dtype == N3D_BF16)
        launch_type<float, __nv_bfloat16>(s, a);
    else if (block_dtype == N3D_F16)
        launch_type<float, __half>(s, a);
    else
        launch_type<float, float>(s, a);
}

}  // namespace n3d
