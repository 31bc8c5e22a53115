// Rotary positions of queries and keys, forward and transposed (n3d_rope).
//
// The pair i of a head at position p turns by p f_i.  The plan holds f_i / 2 pi as a
// 64-bit fraction of a turn, so position * turns[i] modulo 2^64 is the phase without any
// rounding that grows with the position; its top 32 bits (2^-32 of a turn) go through
// sincospi, whose argument needs no reduction.  The transposed rotation negates the sine.
//
// Bound: memory (every element is read and written once, 3 FLOP per element).  A block
// takes a few tokens, evaluates their sines and cosines once into shared memory, and all
// heads of all tensors read them there: per token the trigonometry is rotary_dim / 2
// evaluations against heads * head_dim elements moved.  One launch serves q and k.
//
// A unit is one 16-byte word of each half of the rotary part (half layout), one word of
// it (interleaved), or one word that is copied; a thread keeps its word and walks (token,
// head) rows, so neighbouring threads touch neighbouring words of a head.  Words that turn
// and words that are copied share their loads and stores; the sines are read from shared
// memory 16 bytes a thread without bank conflicts.  A rotary part that is not whole words
// takes the same walk with single pairs, and single elements up to the next word; strides
// or pointers that are not, with single elements throughout.
//
// Measured on a B200: 394 MB of fp32 (128 x 376 tokens, 16 heads of 64) in 64 us, 6.2 TB/s;
// 615 MB of fp16 (30001 tokens, 40 heads of 128, half of each turned, interleaved) in 107 us,
// 5.8 TB/s; 197 MB of bf16 in 41 us, 4.8 TB/s.

#include <algorithm>
#include <climits>

#include "n3d_device.cuh"
#include "train.h"
#include "train_types.cuh"

namespace n3d {

namespace {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 32;  // per block

struct Token {
    long long x[2], y[2], pos;  // element offsets in each tensor, position
};

template <class T, int VEC, bool HALF>
__global__ void __launch_bounds__(THREADS)
    rope_kernel(const __grid_constant__ RopeArgs a, const __grid_constant__ n3d_rope_plan plan, int tile, int wide) {
    // [tile][rotary_dim / 2]: m cos, m sin; two pairs of each word side by side, then the next two of each, so
    // that neighbouring threads read neighbouring 16 bytes
    extern __shared__ float4 trig4[];
    constexpr int PAIRS = HALF ? VEC : VEC == 1 ? 1 : VEC / 2;  // of a unit
    __shared__ Token tok[MAX_TOKENS];
    griddep_wait();
    griddep_launch_dependents();
    const int half = a.rotary_dim / 2;
    const long long t0 = (long long)blockIdx.x * tile;
    const int nt = (int)min((long long)tile, a.tokens - t0);
    if (threadIdx.x < nt) {
        const long long token = t0 + threadIdx.x, seq = token / a.rows, row = token - seq * a.rows;
        Token o;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            o.x[i] = seq * a.x[i].seq + row * a.x[i].row;
            o.y[i] = seq * a.y[i].seq + row * a.y[i].row;
        }
        o.pos = a.positions ? (long long)a.positions[token] : a.first + row;
        tok[threadIdx.x] = o;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nt * half; i += THREADS) {
        const int t = i / half, k = i - t * half;
        const uint64_t phase = (uint64_t)tok[t].pos * plan.turns[k];
        float sn, cs;
        sincospif((float)(int)(uint32_t)(phase >> 32) * 4.656612873077393e-10f, &sn, &cs);  // 2^-31: half turns
        const int u = k / PAIRS, e = k % PAIRS;
        const int at = PAIRS == 1 ? k : (e / 2 * (half / PAIRS) + u) * 2 + e % 2;
        reinterpret_cast<float2*>(trig4)[t * half + at] = make_float2(cs * a.factor, (a.transpose ? -sn : sn) * a.factor);
    }
    __syncthreads();

    // words (pairs of words) that turn, then those that are copied; single pairs are followed by single
    // elements up to the first 16-byte boundary and by whole words where the tensors allow (`wide`)
    constexpr int WORD = 16 / (int)sizeof(T);
    const int turned = half / PAIRS, rest = a.head_dim - a.rotary_dim;
    const int single = VEC > 1 ? 0 : wide ? min(rest, (WORD - a.rotary_dim % WORD) % WORD) : rest;
    const int words = turned + single + (rest - single) / (VEC > 1 ? VEC : WORD);
    const int lanes = THREADS / words;  // (token, head) rows a block walks at a time
    const int w = threadIdx.x % words, lane = threadIdx.x / words;
    if (lane >= lanes) return;
    const bool turns = w < turned;
    // where this thread's word is (VEC > 1, interleaved: turned and copied words alike)
    const int i1 = w - turned;
    const int ca = turns ? (HALF ? w * VEC : VEC == 1 ? 2 * w : w * VEC)
                         : a.rotary_dim + (i1 < single ? i1 : single + (i1 - single) * (VEC > 1 ? VEC : WORD));
    const int cb = HALF ? half + ca : ca + 1;
    for (int which = 0; which < 2; which++) {
        const int heads = which ? a.heads - a.heads0 : a.heads0;
        if (heads == 0 || (!turns && a.in_place[which])) continue;
        const T* const x0 = static_cast<const T*>(a.x[which].p) + ca;
        T* const y0 = static_cast<T*>(a.y[which].p) + ca;
        const long long hx = a.x[which].head, hy = a.y[which].head;
        const int dt = lanes / heads, dh = lanes - dt * heads;
        int t = lane / heads, h = lane - t * heads;
        for (; t < nt; t += dt, h += dh) {
            if (h >= heads) {
                h -= heads;
                if (++t >= nt) break;
            }
            const T* x = x0 + tok[t].x[which] + h * hx;
            T* y = y0 + tok[t].y[which] + h * hy;
            if constexpr (VEC == 1) {
                if (turns) {
                    const float2 r = reinterpret_cast<const float2*>(trig4)[t * half + w];
                    const float p = to_f32<T>(x[0]), q = to_f32<T>(x[cb - ca]);
                    y[0] = from_f32<T>(p * r.x - q * r.y);
                    y[cb - ca] = from_f32<T>(q * r.x + p * r.y);
                } else if (i1 < single) {
                    y[0] = x[0];
                } else {
                    Vec<T, WORD> v;
                    v.load_rw(x);
                    v.store(y);
                }
            } else {
                Vec<T, VEC> va, vb;
                va.load_rw(x);
                if (turns) {
                    const float4* r4 = trig4 + t * half / 2 + w;
                    float p[VEC];
                    if constexpr (HALF) {
                        vb.load_rw(x + half);
                        float q[VEC];
                        va.get(p);
                        vb.get(q);
#pragma unroll
                        for (int i = 0; i < VEC; i += 2) {
                            const float4 r = r4[i / 2 * turned];
                            const float u = p[i] * r.x - q[i] * r.y, v = p[i + 1] * r.z - q[i + 1] * r.w;
                            q[i] = q[i] * r.x + p[i] * r.y;
                            q[i + 1] = q[i + 1] * r.z + p[i + 1] * r.w;
                            p[i] = u, p[i + 1] = v;
                        }
                        vb.set(q);
                        vb.store(y + half);
                    } else {
                        va.get(p);
#pragma unroll
                        for (int i = 0; i < VEC; i += 4) {
                            const float4 r = r4[i / 4 * turned];
                            const float u = p[i] * r.x - p[i + 1] * r.y, v = p[i + 2] * r.z - p[i + 3] * r.w;
                            p[i + 1] = p[i + 1] * r.x + p[i] * r.y;
                            p[i + 3] = p[i + 3] * r.z + p[i + 2] * r.w;
                            p[i] = u, p[i + 2] = v;
                        }
                    }
                    va.set(p);
                }
                va.store(y);
            }
        }
    }
}

template <class T, int VEC, bool HALF>
void launch(cudaStream_t s, const RopeArgs& a, const n3d_rope_plan& plan, bool wide) {
    const int half = a.rotary_dim / 2, rest = a.head_dim - a.rotary_dim, word = 16 / (int)sizeof(T);
    const int words = VEC == 1 ? half + (wide ? rest / word + 1 : rest) : (HALF ? half : a.rotary_dim) / VEC + rest / VEC;
    // Tokens of a block: about 8 words a thread (128 x 376 tokens of 16 heads in bf16: 41 us, with 16 45 us; 30001 tokens
    // of 40 heads in fp16, half of each copied: 107 us, with 4 130 us), halved while that leaves SMs
    // without four blocks.
    constexpr int UNITS = HALF && VEC > 1 ? 4 : 8;
    int tile = (int)std::clamp<long long>((long long)UNITS * THREADS / ((long long)words * a.heads), 1, MAX_TOKENS);
    while (tile > 1 && (a.tokens + tile - 1) / tile < 4LL * sm_count()) tile /= 2;
    const long long blocks = (a.tokens + tile - 1) / tile;
    if (blocks > INT_MAX) throw Error(13, "n3d_rope: more than 2^31 blocks of tokens");
    launch_pdl(rope_kernel<T, VEC, HALF>, dim3((unsigned)blocks), dim3(THREADS), (size_t)tile * half * sizeof(float2), s,
               a, plan, tile, (int)wide);
}

template <class T>
void launch_type(cudaStream_t s, const RopeArgs& a, const n3d_rope_plan& plan) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const bool half = plan.layout == N3D_ROPE_HALF;
    bool wide = a.head_dim % VEC == 0;  // whole 16-byte words of the tensors, if not of the rotary part
    for (int i = 0; i < 2; i++)
        for (const HeadsView* v : {&a.x[i], &a.y[i]})
            wide = wide && reinterpret_cast<uintptr_t>(v->p) % 16 == 0 && v->seq % VEC == 0 && v->row % VEC == 0 &&
                   v->head % VEC == 0;
    const bool words = wide && (half ? a.rotary_dim / 2 : a.rotary_dim) % VEC == 0;
    if (half)
        words ? launch<T, VEC, true>(s, a, plan, true) : launch<T, 1, true>(s, a, plan, wide);
    else
        words ? launch<T, VEC, false>(s, a, plan, true) : launch<T, 1, false>(s, a, plan, wide);
}

}  // namespace

void launch_rope(cudaStream_t s, const RopeArgs& a, const n3d_rope_plan& plan, int dtype) {
    if (a.tokens <= 0 || a.heads <= 0) return;
    if (dtype == N3D_F32)
        launch_type<float>(s, a, plan);
    else if (dtype == N3D_BF16)
        launch_type<__nv_bfloat16>(s, a, plan);
    else
        launch_type<__half>(s, a, plan);
}

}  // namespace n3d
