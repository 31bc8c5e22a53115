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
// it (interleaved), or one word that is copied; threads walk units with the word index
// fixed, so neighbouring threads touch neighbouring words of a head.  A rotary part that is
// not whole words takes the same walk with single pairs, and single elements up to the
// next word; strides or pointers that are not, with single elements throughout.

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
    extern __shared__ float2 trig[];  // [tile][rotary_dim / 2]: m cos, m sin
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
        trig[i] = make_float2(cs * a.factor, (a.transpose ? -sn : sn) * a.factor);
    }
    __syncthreads();

    // words (pairs of words) that turn, then those that are copied; single pairs are followed by single
    // elements up to the first 16-byte boundary and by whole words where the tensors allow (`wide`)
    constexpr int WORD = 16 / (int)sizeof(T);
    const int turned = (HALF || VEC == 1 ? half : a.rotary_dim) / VEC, rest = a.head_dim - a.rotary_dim;
    const int single = VEC > 1 ? 0 : wide ? min(rest, (WORD - a.rotary_dim % WORD) % WORD) : rest;
    const int words = turned + single + (rest - single) / (VEC > 1 ? VEC : WORD);
    const int lanes = THREADS / words;  // (token, head) rows a block walks at a time
    const int w = threadIdx.x % words;
    int h = threadIdx.x / words, t = 0;
    if (h >= lanes) return;
    t = h / a.heads;
    h -= t * a.heads;
    const int dt = lanes / a.heads, dh = lanes - dt * a.heads;
    const bool turns = w < turned;
    for (; t < nt; t += dt, h += dh) {
        if (h >= a.heads) {
            h -= a.heads;
            if (++t >= nt) break;
        }
        const int which = h >= a.heads0;
        const int hh = which ? h - a.heads0 : h;
        const T* x = static_cast<const T*>(a.x[which].p) + tok[t].x[which] + hh * a.x[which].head;
        T* y = static_cast<T*>(a.y[which].p) + tok[t].y[which] + hh * a.y[which].head;
        if (!turns) {
            if (a.in_place[which]) continue;
            const int i = w - turned;
            if (i < single) {
                y[a.rotary_dim + i] = x[a.rotary_dim + i];
            } else {
                const int c = a.rotary_dim + single + (i - single) * WORD;
                Vec<T, WORD> v;
                v.load_rw(x + c);
                v.store(y + c);
            }
        } else if (HALF || VEC == 1) {
            const int ca = HALF ? w * VEC : 2 * w, cb = HALF ? half + w * VEC : 2 * w + 1;
            Vec<T, VEC> va, vb;
            va.load_rw(x + ca);
            vb.load_rw(x + cb);
            float p[VEC], q[VEC];
            va.get(p);
            vb.get(q);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float2 r = trig[t * half + w * VEC + i];
                const float u = p[i] * r.x - q[i] * r.y;
                q[i] = q[i] * r.x + p[i] * r.y;
                p[i] = u;
            }
            va.set(p);
            vb.set(q);
            va.store(y + ca);
            vb.store(y + cb);
        } else {
            Vec<T, VEC> v;
            v.load_rw(x + w * VEC);
            float p[VEC];
            v.get(p);
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const float2 r = trig[t * half + (w * VEC + i) / 2];
                const float u = p[i] * r.x - p[i + 1] * r.y;
                p[i + 1] = p[i + 1] * r.x + p[i] * r.y;
                p[i] = u;
            }
            v.set(p);
            v.store(y + w * VEC);
        }
    }
}

template <class T, int VEC, bool HALF>
void launch(cudaStream_t s, const RopeArgs& a, const n3d_rope_plan& plan, bool wide) {
    const int half = a.rotary_dim / 2, rest = a.head_dim - a.rotary_dim, word = 16 / (int)sizeof(T);
    const int words = VEC == 1 ? half + (wide ? rest / word + 1 : rest) : (HALF ? half : a.rotary_dim) / VEC + rest / VEC;
    // about 8 units per thread, halved while that leaves SMs without four blocks
    int tile = (int)std::clamp<long long>(8LL * THREADS / ((long long)words * a.heads), 1, MAX_TOKENS);
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
