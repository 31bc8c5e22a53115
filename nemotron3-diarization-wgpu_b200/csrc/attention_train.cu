// Attention with its gradient on the fp32 units (n3d_attention_forward, _backward), for
// tensors that the tensor-core kernels do not take: 16-bit ones whose pointers or strides
// are not whole 16-byte words, or that are broadcast, and fp32 ones of at most 64 query and
// key rows (forward only; the rule and its figures are in attention_train_tc.cu).
//
// With S = scale q k^T and lse from the forward pass, P = exp(S - lse) is computed again:
//   D = sum_d dout out,  dP = dout v^T,  dS = P (dP - D)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
// Three kernels from one body: a block owns 64 "row" tokens, walks 64 "column" tokens at
// a time, forms T1 = A1 B1^T (and T2 = A2 B2^T), turns them into weights and multiplies
// these with the column tiles into accumulators in registers:
//   forward  rows = queries, columns = keys:  S;       out += P v       (running max, sum)
//   dq       rows = queries, columns = keys:  S, dP;   dq += dS k       (also writes D)
//   dkv      rows = keys, columns = queries:  S^T, dP^T;  dk += dS^T q, dv += P^T dout
// dq and dkv each recompute S and dP (seven products instead of five) so that every sum
// is taken in a fixed order without atomics.  Masked pairs are set to zero by a select,
// rows past the lengths are never loaded, so nothing that stands there can enter.
//
// Bound: fp32 FMA issue and shared-memory reads about equally: 256 threads as 16 x 16
// hold 4 x 4 scores (rows 4 ty + i, columns tx + 16 j) and 4 x head_dim / 16 accumulators
// each; one 16-byte shared read feeds 8 FMAs.  Row padding of 16 bytes keeps the column
// reads free of bank conflicts.  Measured on a B200 in fp32: 8 x 256 rows, 8 heads of 64, forward
// 49 us, gradient 155 us; tensor cores take 23 and 43.

#include <climits>

#include "n3d_device.cuh"
#include "train.h"
#include "train_types.cuh"

namespace n3d {

namespace {

constexpr int THREADS = 256, TILE = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
enum Mode { FORWARD, GRAD_Q, GRAD_KV };

template <int HD>
struct Smem {
    static constexpr int LD = HD + 4, LP = TILE + 4;  // row strides of the token and the weight tiles
    static constexpr int TOKENS = TILE * LD, WEIGHTS = TILE * LP;
    static constexpr int BYTES = (4 * TOKENS + 2 * WEIGHTS + 4 * TILE) * 4;
};

// Rows [r0, r0 + 64) of a head, zeros at and past `limit`.
template <class T, int HD>
__device__ __forceinline__ void load_tile(float* dst, const HeadsView& t, int seq, int head, int r0, int limit) {
    const T* p = static_cast<const T*>(t.p) + seq * t.seq + head * t.head;
    for (int i = threadIdx.x; i < TILE * HD; i += THREADS) {
        const int r = i / HD, c = i % HD;
        dst[r * Smem<HD>::LD + c] = r0 + r < limit ? to_f32<T>(p[(long long)(r0 + r) * t.row + c]) : 0.0f;
    }
}

// t[i][j] = row (4 ty + i) of a . row (tx + 16 j) of b
template <int HD>
__device__ __forceinline__ void product(const float* a, const float* b, int ty, int tx, float (&t)[4][4]) {
    constexpr int LD = Smem<HD>::LD;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) t[i][j] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * LD + d);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * LD + d);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                t[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
    }
}

// acc[i][c] += sum over the 64 columns of w[4 ty + i][column] * b[column][elements 4 tx + 64 c ..]
template <int HD>
__device__ __forceinline__ void accumulate(const float* w, const float* b, int ty, int tx, float (&acc)[4][HD / 16]) {
    constexpr int LD = Smem<HD>::LD, LP = Smem<HD>::LP;
#pragma unroll 2
    for (int c = 0; c < TILE; c += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = *reinterpret_cast<const float4*>(w + (4 * ty + i) * LP + c);
#pragma unroll
        for (int cc = 0; cc < 4; cc++)
#pragma unroll
            for (int e = 0; e < HD / 64; e++) {
                const float4 y = *reinterpret_cast<const float4*>(b + (c + cc) * LD + 64 * e + 4 * tx);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float u = cc == 0 ? p[i].x : cc == 1 ? p[i].y : cc == 2 ? p[i].z : p[i].w;
                    acc[i][4 * e] += u * y.x;
                    acc[i][4 * e + 1] += u * y.y;
                    acc[i][4 * e + 2] += u * y.z;
                    acc[i][4 * e + 3] += u * y.w;
                }
            }
    }
}

template <class T, int HD>
__device__ __forceinline__ void store_rows(const HeadsView& t, int seq, int head, int r0, int rows, int ty, int tx,
                                           const float (&acc)[4][HD / 16], const float (&factor)[4]) {
    T* p = static_cast<T*>(t.p) + seq * t.seq + head * t.head;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = r0 + 4 * ty + i;
        if (r >= rows) continue;
#pragma unroll
        for (int c = 0; c < HD / 16; c++)
            p[(long long)r * t.row + 64 * (c / 4) + 4 * tx + c % 4] = from_f32<T>(acc[i][c] * factor[i]);
    }
}

template <class T, int HD, int MODE>
__global__ void __launch_bounds__(THREADS) attention_train_kernel(const __grid_constant__ AttnArgs a, int tiles) {
    using S = Smem<HD>;
    extern __shared__ float4 smem4[];
    float* a1 = reinterpret_cast<float*>(smem4);
    float *a2 = a1 + S::TOKENS, *b1 = a2 + S::TOKENS, *b2 = b1 + S::TOKENS;
    float *w1 = b2 + S::TOKENS, *w2 = w1 + S::WEIGHTS;
    float *col_lse = w2 + S::WEIGHTS, *col_dot = col_lse + TILE, *row_lse = col_dot + TILE, *row_dot = row_lse + TILE;
    griddep_wait();
    griddep_launch_dependents();
    const int heads = MODE == GRAD_KV ? a.k_heads : a.q_heads, group = a.q_heads / a.k_heads;
    const int tile = blockIdx.x % tiles, sh = blockIdx.x / tiles, head = sh % heads, seq = sh / heads;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int r0 = tile * TILE;
    const AttnMask mask(a, seq);
    const float k2 = a.scale * LOG2E;

    float acc1[4][HD / 16] = {}, acc2[4][HD / 16] = {};
    float top[4], sum[4];  // forward: running max (of the scaled exponents) and sum
#pragma unroll
    for (int i = 0; i < 4; i++) top[i] = -INFINITY, sum[i] = 0.0f;

    const int row_len = MODE == GRAD_KV ? mask.k_len : mask.q_len;
    const int r1 = min(r0 + TILE, row_len) - 1;  // last row inside the length
    int c_begin = 0, c_end = 0;
    if (r1 >= r0) {
        c_begin = MODE == GRAD_KV ? mask.first_query(r0) : mask.first_key(r0);
        c_end = MODE == GRAD_KV ? mask.last_query(r1) : mask.last_key(r1);
    }
    if (MODE == GRAD_KV) {
        load_tile<T, HD>(a1, a.k, seq, head, r0, row_len);
        load_tile<T, HD>(a2, a.v, seq, head, r0, row_len);
    } else {
        load_tile<T, HD>(a1, a.q, seq, head, r0, row_len);
    }
    if (MODE == GRAD_Q) {
        load_tile<T, HD>(a2, a.dout, seq, head, r0, row_len);
        load_tile<T, HD>(b1, a.o, seq, head, r0, row_len);
        __syncthreads();
        const long long at = ((long long)seq * a.q_heads + head) * a.q_rows + r0;
        const int r = threadIdx.x / 4;  // four threads of a warp per row
        float d = 0.0f;
#pragma unroll 4
        for (int c = threadIdx.x % 4; c < HD; c += 4) d += a2[r * S::LD + c] * b1[r * S::LD + c];
        d += __shfl_xor_sync(0xffffffffu, d, 1);
        d += __shfl_xor_sync(0xffffffffu, d, 2);
        if (threadIdx.x % 4 == 0) {
            row_dot[r] = d;
            row_lse[r] = INFINITY;
            if (r0 + r < a.q_rows) {
                a.row_dot[at + r] = d;
                const float l = a.lse[at + r];
                if (r0 + r < row_len && l != -INFINITY) row_lse[r] = l * LOG2E;
            }
        }
    }

    for (int g = 0; g < (MODE == GRAD_KV ? group : 1); g++) {
        const int col_head = MODE == GRAD_KV ? head * group + g : head / group;
        for (int c0 = c_begin / TILE * TILE; c0 < c_end; c0 += TILE) {
            __syncthreads();  // the previous tiles and weights are read
            if (MODE == GRAD_KV) {
                load_tile<T, HD>(b1, a.q, seq, col_head, c0, mask.q_len);
                load_tile<T, HD>(b2, a.dout, seq, col_head, c0, mask.q_len);
                if (threadIdx.x < TILE) {
                    const int i = c0 + threadIdx.x;
                    const long long at = ((long long)seq * a.q_heads + col_head) * a.q_rows + i;
                    const float l = i < mask.q_len ? a.lse[at] : -INFINITY;
                    col_lse[threadIdx.x] = l == -INFINITY ? INFINITY : l * LOG2E;
                    col_dot[threadIdx.x] = i < mask.q_len ? a.row_dot[at] : 0.0f;
                }
            } else {
                load_tile<T, HD>(b1, a.k, seq, col_head, c0, mask.k_len);
                load_tile<T, HD>(b2, a.v, seq, col_head, c0, mask.k_len);
            }
            __syncthreads();
            float t1[4][4], t2[4][4];
            product<HD>(a1, b1, ty, tx, t1);
            if (MODE != FORWARD) product<HD>(a2, b2, ty, tx, t2);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = r0 + 4 * ty + i;
                const int lo = MODE == GRAD_KV ? mask.first_query(r) : mask.first_key(r);
                const int hi = r >= row_len ? 0 : MODE == GRAD_KV ? mask.last_query(r) : mask.last_key(r);
                if (MODE == FORWARD) {
                    float m = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int c = c0 + tx + 16 * j;
                        t1[i][j] = c >= lo && c < hi ? t1[i][j] * k2 : -INFINITY;
                        m = fmaxf(m, t1[i][j]);
                    }
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    m = fmaxf(m, top[i]);
                    const float base = m == -INFINITY ? 0.0f : m;  // nothing seen yet: exponents stay -inf
                    const float keep = exp2f(top[i] - base);
                    top[i] = m;
                    float s = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float p = exp2f(t1[i][j] - base);
                        w1[(4 * ty + i) * S::LP + tx + 16 * j] = p;
                        s += p;
                    }
                    sum[i] = sum[i] * keep + s;
#pragma unroll
                    for (int c = 0; c < HD / 16; c++) acc1[i][c] *= keep;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int cc = tx + 16 * j, c = c0 + cc;
                        const float lse = MODE == GRAD_KV ? col_lse[cc] : row_lse[4 * ty + i];
                        const float dot = MODE == GRAD_KV ? col_dot[cc] : row_dot[4 * ty + i];
                        const bool seen = c >= lo && c < hi;
                        // (held at 1 where the statistics' rounding passes the exponent's: huge scores)
                        const float p = seen ? exp2f(fminf(t1[i][j] * k2 - lse, 0.0f)) : 0.0f;
                        if (MODE == GRAD_KV) w2[(4 * ty + i) * S::LP + cc] = p;
                        w1[(4 * ty + i) * S::LP + cc] = seen ? p * (t2[i][j] - dot) : 0.0f;
                    }
                }
            }
            __syncthreads();
            accumulate<HD>(w1, MODE == FORWARD ? b2 : b1, ty, tx, acc1);
            if (MODE == GRAD_KV) accumulate<HD>(w2, b2, ty, tx, acc2);
        }
    }

    float factor[4];
#pragma unroll
    for (int i = 0; i < 4; i++) factor[i] = a.scale;
    if (MODE == FORWARD) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
            const int r = r0 + 4 * ty + i;
            factor[i] = sum[i] > 0.0f ? 1.0f / sum[i] : sum[i] == 0.0f ? 0.0f : NAN;
            if (a.lse && tx == 0 && r < a.q_rows)
                a.lse[((long long)seq * a.q_heads + head) * a.q_rows + r] =
                    sum[i] == 0.0f ? -INFINITY : (top[i] + log2f(sum[i])) * LN2;
        }
        store_rows<T, HD>(a.o, seq, head, r0, a.q_rows, ty, tx, acc1, factor);
    } else if (MODE == GRAD_Q) {
        store_rows<T, HD>(a.dq, seq, head, r0, a.q_rows, ty, tx, acc1, factor);
    } else {
        store_rows<T, HD>(a.dk, seq, head, r0, a.k_rows, ty, tx, acc1, factor);
#pragma unroll
        for (int i = 0; i < 4; i++) factor[i] = 1.0f;
        store_rows<T, HD>(a.dv, seq, head, r0, a.k_rows, ty, tx, acc2, factor);
    }
}

template <class T, int HD, int MODE>
void launch(cudaStream_t s, const AttnArgs& a) {
    static std::atomic<unsigned long long> attr{0};
    once_per_device(attr, [] {
        N3D_CUDA(cudaFuncSetAttribute(attention_train_kernel<T, HD, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      Smem<HD>::BYTES));
    });
    const int rows = MODE == GRAD_KV ? a.k_rows : a.q_rows, heads = MODE == GRAD_KV ? a.k_heads : a.q_heads;
    const int tiles = (rows + TILE - 1) / TILE;
    const long long blocks = (long long)tiles * heads * a.seqs;
    if (blocks > INT_MAX) throw Error(13, "attention: more than 2^31 tiles");
    if (blocks == 0) return;
    launch_pdl(attention_train_kernel<T, HD, MODE>, dim3((unsigned)blocks), dim3(THREADS), Smem<HD>::BYTES, s, a, tiles);
}

template <class T, int HD>
void launch_modes(cudaStream_t s, const AttnArgs& a, bool backward) {
    if (!backward) return launch<T, HD, FORWARD>(s, a);
    launch<T, HD, GRAD_Q>(s, a);
    launch<T, HD, GRAD_KV>(s, a);
}
template <class T>
void launch_dim(cudaStream_t s, const AttnArgs& a, bool backward) {
    a.head_dim == 64 ? launch_modes<T, 64>(s, a, backward) : launch_modes<T, 128>(s, a, backward);
}
void launch_type(cudaStream_t s, const AttnArgs& a, int dtype, bool backward) {
    if (attention_tc_fits(a, dtype, backward)) return launch_attention_train_tc(s, a, dtype, backward);
    if (dtype == N3D_F32)
        launch_dim<float>(s, a, backward);
    else if (dtype == N3D_BF16)
        launch_dim<__nv_bfloat16>(s, a, backward);
    else
        launch_dim<__half>(s, a, backward);
}

}  // namespace

void launch_attention_forward(cudaStream_t s, const AttnArgs& a, int dtype) { launch_type(s, a, dtype, false); }
void launch_attention_backward(cudaStream_t s, const AttnArgs& a, int dtype) { launch_type(s, a, dtype, true); }

}  // namespace n3d
