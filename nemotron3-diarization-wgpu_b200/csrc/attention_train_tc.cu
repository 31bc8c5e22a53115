// Attention with its gradient on the sm_100a tensor cores (tcgen05, kind::f16) for bf16
// and fp16 tensors (n3d_attention_forward, _backward); the formulas are those of
// attention_train.cu, and so are the three passes from one body:
//   forward  rows = queries, columns = keys:  T1 = q k^T;                  out += P v
//   dq       rows = queries, columns = keys:  T1 = q k^T, T2 = dout v^T;   dq += dS k
//   dkv      rows = keys, columns = queries:  T1 = k q^T, T2 = v dout^T;   dk += dS^T q, dv += P^T dout
//
// A block works on items of 128 rows of a head (TMEM lanes, one softmax thread each) and walks
// blocks of 64 columns.  When an item's loads are under way it takes the next one over from
// the grid by cluster launch control, so that launch, set-up and epilogue overlap (windows of
// 384 rows: forward 97 us with a block per item, 75 so).  The column tiles are K-major
// operands of T1 and T2 in shared memory; the weights (P, dS) go back to TMEM as the 16-bit
// A operand of the second product, over scores that are read, and its B operand is the same
// column tile read with the token index as K (MN-major), so no tile is stored twice or
// transposed.  The row tiles are T's A operands: in TMEM where they fit and pay (ROW_TMEM),
// else in shared memory.  Nothing of size rows x columns leaves the SM.
//   warp 0      items; TMA: the row tiles, the column tiles through a ring of stages
//   warp 1      TMEM owner; issues T of block g once its score buffer is free (see EARLY)
//   warp 2      issues the second products (with both kinds on one thread the gradient of 2 x 4096 rows,
//               16 heads of 128, took 1092 us against 946; a thread for each of the four products of
//               dkv gains nothing more)
//   warps 3..   softmax groups of 4 warps, one thread per row; NWG column blocks are in work at a time
// head_dim 64: one group and two blocks per SM, which interleave (256 TMEM columns each);
// head_dim 128: one block per SM with two groups on alternating column blocks (forward:
// each with its own running maximum, sum and accumulator, joined at the end).
//
// dq and dkv both recompute T1 and T2: seven products where a kernel that adds dq
// atomically needs five, but each sum is taken in one accumulator in a fixed order, and
// no fp32 copy of dq passes through memory.  dq runs first and leaves -lse log2 e and -D
// of each row for dkv, where they belong to columns and come through the ring.
//
// fp16: P is kept times 2^7 (forward, P <= 2^8 there) or 2^10 (dkv), and dS times 2^3 /
// |dout row| (dq) or over the largest |dout row| of the head group (dkv), as powers of
// two, so that small weights and gradients keep fp16's precision.  dS_j = P_j (1 - P_j) dout . (v_j - o'), o' the
// mean of the other rows of v by their weights, so |dS| <= |dout row| max |v row| / 2, and times up to 16 /
// |dout row| it stays below 2^15 while |v row| < 4096.  (In dkv the rows with the least dout lose bits: where
// P |dout row| |v row| is below 2^-16 of the largest |dout row|, dS is subnormal.)
//
// fp32: every operand is a pair h + l of fp16 arrays (attention_train_split.cu), each row of it in a unit
// of its own, a power of two; the weights are split in the softmax, and each product is l h + h l + h h.
// Scores and T2 are multiplied by the units of their row and column; a weight by the unit of the column
// that the second product multiplies it with, and then by a power of two of its own row that
// brings the row's largest weight of the block into [64, 128).  So each row of each operand, and each row of
// weights, keeps 22 bits however small it is beside others, and no sequence depends on the others of its batch.
// The tensor cores' fp32 accumulators truncate: about 2^-26 of the accumulator per MMA, always
// towards zero, which 12 MMAs a block carry to 1.5e-5 at 4096 rows.  So an accumulator takes two blocks, the
// small products of each first, and is then added to a sum that is rounded to nearest (more
// TMEM, or the output tensor), which also takes it out of its row's unit.  The second block of two keeps the
// first one's unit unless its own weights do not fit there.
//
// Bound, from clock stamps in every role: at head_dim 128 in forward and dq the thread that
// issues T, whose block of 8 or 16 MMAs takes 300 - 570 clocks and each wait, passed at once,
// another 110 - 170 (tensor pipe 46 - 48 % busy); in dkv the chain of a score buffer, softmax 1500 -
// 1800, second products 500 - 800, T2 450.  At head_dim 64 the softmax threads: in forward they work
// without a pause, in the gradients they wait for T (750 of 1850 clocks in dq, 850 of 2900 in dkv) while
// the SM's other block computes.  Measured on a B200: 128 windows of 384 rows, 8 heads of 64, bf16,
// forward 74 us and gradient 253 us (520 and 535 executed TFLOP/s); 2 x 4096 rows, 16 heads of 128, 255
// and 873 us (1080 and 1100); the same causal with 4 key heads 136 and 497 us.
//
// Rows past a sequence's length: TMA fills what lies past the tensor with zeros, and the
// T warp overwrites what lies past the length with zeros before a tile is used, so
// nothing that stands there enters a product.  Pairs that the mask hides are cleared by a
// select.  Every wait is bounded; an expired wait records its site and the block returns.
// Each barrier is waited for at most one phase behind (argued at the waits).

#include <algorithm>
#include <climits>
#include <type_traits>

#include "n3d_device.cuh"
#include "train.h"
#include "train_types.cuh"

namespace n3d {

namespace {

enum Mode { FORWARD, GRAD_Q, GRAD_KV };
constexpr int ROWS = 128, COLS = 64;
constexpr int BOX = 64 * 128;  // a TMA box: 64 rows of 64 elements
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_LOG2 = 8.0f;  // forward: raise the running maximum when exponents would exceed 2^8
constexpr float FAR = 32768.0f;  // exponents whose rounding, 2^-9, is no longer small
constexpr int DEV_TIMEOUT_ATTN_TRAIN = 7;

// PARTS: 1 for 16-bit tensors, 2 for fp32 tensors as fp16 pairs h + l.
template <int HD, int MODE, int PARTS>
struct Cfg {
    static constexpr bool GRAD = MODE != FORWARD;
    static constexpr bool SMALL = HD == 64 && PARTS == 1;   // two blocks fit an SM
    static constexpr bool PAIR = PARTS == 2;
    // column blocks in softmax at a time (an fp32 forward pass of head_dim 128 has TMEM for one)
    static constexpr int NWG = SMALL || (PAIR && HD == 128 && MODE == FORWARD) ? 1 : 2;
    // Row tiles as TMEM operands.  2 x 4096 rows, 16 heads of 128, us with and without: forward 265 and 272, gradient
    // (dq) 931 and 959; 128 windows of 384 rows, 8 heads of 64: gradient 262 and 268, but forward 78.7 and
    // 75.7 (the copy is on the path of every item of six blocks).  dkv's accumulators leave no room, nor do pairs.
    static constexpr bool ROW_TMEM = !PAIR && (MODE == GRAD_Q || (MODE == FORWARD && HD == 128));
    // Score buffers, as many as TMEM holds where that pays.  Forward of 128: a third took 312 us to 265, with the
    // row tiles' move; forward of pairs, 2 x 4096 rows, 16 heads of 64: two 852 us, three 766, four 693 (of 128:
    // no change); dq of pairs, 64 heads of 501 rows of 64: a third takes the gradient from 109 to 107.
    static constexpr int NBUF = PAIR && HD == 64 && MODE != GRAD_KV ? (MODE == FORWARD ? 4 : 3) : MODE != FORWARD ? NWG : ROW_TMEM ? 3 : 2;
    // gradients whose weights all lie over T2: T1 of the buffer's next block need not wait for the products that
    // read them
    static constexpr bool EARLY = GRAD && !(PAIR && MODE == GRAD_KV);
    static constexpr int SOFTMAX = 3;                       // first softmax warp
    static constexpr int THREADS = 32 * SOFTMAX + 128 * NWG, PER_SM = SMALL ? 2 : 1;
    static constexpr int RTILE = ROWS * HD * 2 * PARTS, CTILE = COLS * HD * 2 * PARTS;  // bytes
    // 64 x (-lse log2 e), 64 x (-D), pairs: the units of q and dout; pairs otherwise: those of k and v
    static constexpr int STATS = MODE == GRAD_KV ? (PAIR ? kSplitStat : 128) * 4 : PAIR ? kKeyStat * 4 : 0;
    static constexpr int STAT_LD = PARTS == 1 ? 128 : kSplitStat;         // floats of a block of 64 rows
    static constexpr int STAGE = 2 * CTILE + 1024 * (STATS > 0);
    static constexpr int ROW_BYTES = (GRAD ? 2 : 1) * RTILE;
    // floats of the groups' row statistics (double-buffered by item)
    static constexpr int JOIN = MODE == FORWARD ? (NWG > 1 ? (4 + 4 * PAIR) * 128 : 4) : PAIR ? 2 * 128 : 4;
    // pairs, gradients: the rows' units of the weights, from the group of an even block to that of the next
    // (double-buffered by pair of blocks)
    static constexpr int UNITS = PAIR && GRAD ? 4 * 128 : 0;
    // barriers, items, the TMEM slot, the statistics, and slack to align the tiles to 1024 bytes
    static constexpr int REST = 704 + 2 * JOIN * 4 + UNITS * 4 + 1024;
    static constexpr int ROOM = 226 * 1024 / PER_SM - REST;
    // Row tiles of two items, so that the next one's load during this one's work, where that leaves enough
    // stages.  Gradient of 64 windows of 384 rows of 64: 155 us with two and two, 174 with one and four;
    // of 2 x 4096 rows of 128, with one block per SM: 1091 against 958.
    static constexpr int RB = (ROOM - 2 * ROW_BYTES) / STAGE >= (SMALL ? 2 : 3) ? 2 : 1;
    static constexpr int NST = (ROOM - RB * ROW_BYTES) / STAGE > 4 ? 4 : (ROOM - RB * ROW_BYTES) / STAGE;
    static constexpr int SMEM = RB * ROW_BYTES + NST * STAGE + REST;
    static constexpr uint32_t TBUF = GRAD ? 128 : 64;                     // TMEM columns of a score buffer
    static constexpr uint32_t ACC = NBUF * TBUF;                          // first accumulator
    static constexpr int NACC = MODE == FORWARD ? NWG : MODE == GRAD_Q ? 1 : 2;
    // pairs: the accumulators are added up after them (see the head of the file); dk and dv
    // of head_dim 128 are added up in the output tensors, for which there is no TMEM
    static constexpr bool SUM = PAIR, SUM_OUT = PAIR && HD == 128 && MODE == GRAD_KV;
    static constexpr uint32_t ROWT = ACC + (SUM && !SUM_OUT ? 2 : 1) * NACC * HD;  // first column of the row tiles
    static constexpr uint32_t TMEM_COLS = SMALL ? 256 : 512;
    static_assert(ROWT + (ROW_TMEM ? (GRAD ? 2 : 1) * HD / 2 : 0) <= TMEM_COLS && PER_SM * TMEM_COLS <= 512, "TMEM");
    static_assert(NST >= 1 && (SMEM + 1024) * PER_SM <= 228 * 1024, "shared memory");
};

// Instruction descriptor of kind::f16 with fp32 accumulators, M = 128; B K-major, or
// MN-major (token index as K); A negated for a negative score scale.
template <class T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn, bool negate_a = false) {
    const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(negate_a) << 13) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
// Descriptor of an MN-major B tile: boxes of 64 d-elements (128-byte swizzled rows, one
// row per token); 8-token groups 1024 B apart (SBO), boxes BOX apart (LBO).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(BOX >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int d, int row, int head,
                                            int seq) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
            "r"(smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(d), "r"(row), "r"(head), "r"(seq)
        : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int d, int row, int head,
                                             int seq) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map),
                 "r"(d), "r"(row), "r"(head), "r"(seq), "r"(smem_u32(src))
                 : "memory");
}
// Untiled copy of `bytes` (a multiple of 16, both addresses 16-byte aligned).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, int bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
// Cluster launch control: takes the next block of the grid that has not started, if any, over
// from the scheduler; the answer (16 bytes) arrives on `bar`.
__device__ __forceinline__ void try_cancel(void* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(answer)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// The block taken over, -1 if none was left.
__device__ __forceinline__ int cancelled_block(const void* answer) {
    uint32_t ok, x = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t.reg .b32 y, z, w;\n\t"
        "ld.shared.b128 a, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, a;\n\t}"
        : "=r"(ok), "=r"(x)
        : "r"(smem_u32(answer))
        : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    return ok ? (int)x : -1;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 16 TMEM columns of this thread's lane from 32-bit words; completes with tmem_wait_st().
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t* v) {
    static_assert(N == 8 || N == 16, "8 or 16 columns");
    N == 8 ? tmem_st8(taddr, v) : tmem_st16(taddr, v);
}
// 16 columns at each of two places of this thread's lane: both loads, one wait.
__device__ __forceinline__ void tmem_ld_pair(uint32_t a, uint32_t b, float* x, float* y) {
    uint32_t r[32];
#pragma unroll
    for (int h = 0; h < 2; h++)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[16 * h + 0]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]), "=r"(r[16 * h + 4]),
              "=r"(r[16 * h + 5]), "=r"(r[16 * h + 6]), "=r"(r[16 * h + 7]), "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]),
              "=r"(r[16 * h + 10]), "=r"(r[16 * h + 11]), "=r"(r[16 * h + 12]), "=r"(r[16 * h + 13]),
              "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
            : "r"(h ? b : a));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    reg_fence16(r);
    reg_fence16(r + 16);
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = __uint_as_float(r[i]), y[i] = __uint_as_float(r[16 + i]);
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^-floor(log2 x) for a positive normal x, 1 otherwise
__device__ __forceinline__ float inverse_power(float x) {
    const int e = (__float_as_int(x) >> 23) & 255;
    return x > 0.0f && e > 0 && e < 254 ? __int_as_float((254 - e) << 23) : 1.0f;
}

// ln(l 2^(m k2 - shift)) for a row sum l >= 0: -inf for an empty row.  The exponent and the logarithm
// of the mantissa are added in fp64, so that the result carries little more than its own rounding.
__device__ __forceinline__ float row_lse(float l, float m, float k2, float shift) {
    if (l == 0.0f) return -INFINITY;
    if (!(l < INFINITY)) return l;
    const int bits = __float_as_int(l);
    const float mantissa = __int_as_float((bits & 0x7fffff) | 0x3f800000);
    const double t = (double)m * (double)k2 + ((double)((bits >> 23) - 127) - (double)shift) + (double)log2f(mantissa);
    return (float)(t * 0.6931471805599453);
}
// Four floats of shared memory, not moved ahead of what stands before it (which would hold registers).
__device__ __forceinline__ float4 lds4(const float4* p) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_u32(p)));
    return v;
}
// -lse log2 e of a row for the gradient.  Beyond 2^18 its rounding (here, and lse's own) matters: at 2^30 P would come out as
// any power of two up to 2^128, and the gradients infinite.  There it is moved by a little more than that
// rounding, so that P <= 1.  (Holding each exponent at 0 instead, as pairs do, took the gradient of 64 windows of
// 377 rows of 64 in fp16 from 162 us to 167, a test for such rows to 165.)
__device__ __forceinline__ float row_nlse(float lse) {
    const float n = -lse * LOG2E;
    return fabsf(n) > 262144.0f ? n - fabsf(n) * 2.384185791015625e-7f : n;  // 2^-22
}
// Pairs: the power of two that brings a row's largest weight w into [64, 128); 1 if there is none.  (Held below
// 2^126, so that its inverse is normal too.)
__device__ __forceinline__ float weight_unit(float w) {
    return w > 0.0f && w < INFINITY ? __int_as_float(min(253, 260 - (__float_as_int(w) >> 23)) << 23) : 1.0f;
}
constexpr float MAX_WEIGHT = 32768.0f;  // that a row's unit may bring a weight to
// The largest of sixteen magnitudes and m.
__device__ __forceinline__ float max16(const float* x, float m) {
    float a = fabsf(x[0]), b = fabsf(x[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 4) {
        a = max3f(a, fabsf(x[i]), fabsf(x[i + 1]));
        if (i + 2 < 16) b = max3f(b, fabsf(x[i + 2]), fabsf(x[i + 3]));
    }
    return max3f(m, a, b);
}

// Both waits, tested one behind the other before either's result is used: a wait that passes at once costs the issuing
// warps 110 - 170 clocks, which two in a row would pay twice for every block.
__device__ __forceinline__ bool wait_both(uint64_t* a, uint32_t phase_a, uint64_t* b, uint32_t phase_b, int* err) {
    const bool pa = mbar_try_wait(a, phase_a), pb = mbar_try_wait(b, phase_b);
    return (pa || mbar_wait(a, phase_a, err, DEV_TIMEOUT_ATTN_TRAIN)) && (pb || mbar_wait(b, phase_b, err, DEV_TIMEOUT_ATTN_TRAIN));
}

struct TcMaps {
    CUtensorMap q, k, v, dout;       // loads, 64-row boxes
    CUtensorMap out, dq, dk, dv;     // stores, 32-row boxes
};
struct TcArgs {
    AttnArgs a;
    int tiles;         // row tiles of a head
    int run;           // heads whose tiles are interleaved
    int ascending;     // which end of a one-sided window is open: 1 if keys before the query
    float k2, factor;  // |scale| log2 e; the scale of dq and dk
    int negate;        // scale < 0
    float* stats;      // [seqs * q_heads][q tiles][2][-lse log2 e: 64 | -D: 64 (| pairs: units of q: 64 | of dout: 64)]
    float* norms;      // [seqs * q_heads][q tiles]: the largest |dout row|
    const float* key_stats;  // pairs: [seqs * k_heads][k tiles][units of k: 64 | of v: 64]
    int q_tiles, k_tiles;    // of 128 query rows, of 64 key rows
};

// T: the type of the MMA operands; tensors are of type T (PARTS 1) or fp32 (PARTS 2, T = fp16).
// What a block works on: 128 rows of a head and the column blocks they see.
struct Item {
    int seq, head, r0, row_len, col_len;
    int c_begin, per_head, nblk;  // first column block, blocks of one column head, blocks
    int full_lo, full_hi;         // columns that every live row sees
    int valid, pad;
};
static_assert(sizeof(Item) == 48, "two items in 96 bytes");

template <class T, int HD, int MODE, int PARTS>
__global__ void __launch_bounds__(Cfg<HD, MODE, PARTS>::THREADS, Cfg<HD, MODE, PARTS>::PER_SM)
    attention_train_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcArgs args) {
    using C = Cfg<HD, MODE, PARTS>;
    constexpr bool F16 = std::is_same<T, __half>::value, PAIR = PARTS == 2;
    constexpr int RPART = ROWS * HD * 2, CPART = COLS * HD * 2;  // bytes of one part of a tile
    constexpr int NWG = C::NWG, NBUF = C::NBUF, NST = C::NST;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* rows = smem;                        // RB x (rows 1 | rows 2)
    uint8_t* ring = smem + C::RB * C::ROW_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NST * C::STAGE);
    uint64_t* r_full = bars;               // RB: row tiles of loaded item n landed (buffer n % RB)
    uint64_t* r_free = r_full + 2;         // RB: their item's outputs have left the buffer (every softmax warp)
    uint64_t* c_full = r_free + 2;         // NST: the column tiles of block g landed (stage g % NST)
    uint64_t* c_empty = c_full + 4;        // NST: block g's second products completed
    uint64_t* t_full = c_empty + 4;        // NBUF: T of block g completed (buffer g % NBUF)
    uint64_t* p_full = t_full + 4;         // NBUF: weights of block g written
    uint64_t* acc_done = p_full + 4;       // NBUF: second products of block g completed
    uint64_t* acc_free = acc_done + 4;     // NWG (pairs): the accumulator is added to its sum (4 warps)
    uint64_t* all_done = acc_free + 2;     // 1: phase n = the last product of loaded item n completed
    uint64_t* acc_read = all_done + 1;     // 1: phase n = its accumulators are read (every softmax warp)
    uint64_t* rows_in = acc_read + 1;      // 1: phase n = its row tiles are in TMEM (every softmax warp)
    uint64_t* item_full = rows_in + 1;     // 2: item k is known (slot k % 2)
    uint64_t* item_empty = item_full + 2;  // 2: item k was read by every other warp
    uint64_t* answered = item_empty + 2;   // 1: the scheduler's answer arrived
    uint64_t* unit_set = answered + 1;     // 2 (pairs, gradients): the units of pair of blocks x are known (slot x % 2)
    static_assert(NST <= 4 && NBUF <= 4 && NWG <= 2 && C::RB <= 2, "barriers");
    Item* items = reinterpret_cast<Item*>(bars + 36);  // 2
    uint8_t* answer = reinterpret_cast<uint8_t*>(bars + 48);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 50);
    float* joins = reinterpret_cast<float*>(bars + 52);  // 2 x JOIN
    float* units = joins + 2 * C::JOIN;                  // UNITS

    // The reduction tells the compiler that a value is the same in the warp, which keeps what the issuing warps
    // derive from it in uniform registers, where MMAs take their operands from.
    auto uniform = [](int x) { return (int)__reduce_max_sync(0xffffffffu, x); };
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (warp == 0 && lane == 0) {
        for (int i = 0; i < C::RB; i++) mbar_init(&r_full[i], 1), mbar_init(&r_free[i], 4 * NWG);
        for (int i = 0; i < NST; i++) mbar_init(&c_full[i], 1), mbar_init(&c_empty[i], 1);
        for (int i = 0; i < NBUF; i++)
            mbar_init(&t_full[i], 1), mbar_init(&p_full[i], 4), mbar_init(&acc_done[i], 1);
        for (int i = 0; i < NWG; i++) mbar_init(&acc_free[i], 4);
        mbar_init(all_done, 1);
        mbar_init(acc_read, 4 * NWG);
        mbar_init(rows_in, 4 * NWG);
        for (int i = 0; i < 2; i++) mbar_init(&item_full[i], 1), mbar_init(&item_empty[i], 2 + 4 * NWG);
        mbar_init(answered, 1);
        for (int i = 0; i < 2; i++) mbar_init(&unit_set[i], 4);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, C::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    griddep_wait();
    griddep_launch_dependents();

    const AttnArgs& a = args.a;
    int* const err = a.err;
    const int heads = MODE == GRAD_KV ? a.k_heads : a.q_heads, group = a.q_heads / a.k_heads;
    const int row_cap = MODE == GRAD_KV ? a.k_rows : a.q_rows, col_cap = MODE == GRAD_KV ? a.q_rows : a.k_rows;
    auto first_col = [&](const AttnMask& mask, int r) { return MODE == GRAD_KV ? mask.first_query(r) : mask.first_key(r); };
    auto last_col = [&](const AttnMask& mask, int r) { return MODE == GRAD_KV ? mask.last_query(r) : mask.last_key(r); };
    auto col0 = [&](const Item& it, int g) { return (it.c_begin + (MODE == GRAD_KV ? g % it.per_head : g)) * COLS; };
    auto col_head = [&](const Item& it, int g) {
        return MODE == GRAD_KV ? it.head * group + g / it.per_head : it.head / group;
    };
    // item k for every warp but the first: false after the last one, or when a wait expired
    auto next_item = [&](int k, Item& it) {
        // (phase k / 2 of its slot: the next needs this warp's arrival below)
        if (!__all_sync(0xffffffffu, mbar_wait(&item_full[k & 1], (k >> 1) & 1, err, DEV_TIMEOUT_ATTN_TRAIN))) return false;
        it = items[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[k & 1]);
        return it.valid != 0;
    };
    // the same for an issuing warp
    auto next_uniform = [&](int k, Item& it) {
        const bool more = next_item(k, it);
        it.r0 = uniform(it.r0), it.row_len = uniform(it.row_len), it.col_len = uniform(it.col_len);
        it.c_begin = uniform(it.c_begin), it.per_head = uniform(it.per_head), it.nblk = uniform(it.nblk);
        return (bool)__all_sync(0xffffffffu, more);
    };

    // Every role walks the same items; g counts the column blocks and n the items with any, over all of them:
    // buffers, stages and phases go by these numbers.
    if (warp == 0) {
        if (lane == 0) {
            const CUtensorMap* rm1 = MODE == GRAD_KV ? &maps.k : &maps.q;
            const CUtensorMap* rm2 = MODE == GRAD_KV ? &maps.v : &maps.dout;
            const CUtensorMap* cm1 = MODE == GRAD_KV ? &maps.q : &maps.k;
            const CUtensorMap* cm2 = MODE == GRAD_KV ? &maps.dout : &maps.v;
            bool ok = true;
            int gt = 0, n = 0, block = blockIdx.x;
            for (int k = 0; ok; k++) {
                // ---- item k: heads in runs of args.run; within a run the same tile of every head, then the next
                // tile.  Under a one-sided window the tiles with the most columns go first (the last query
                // tiles see the most keys, the first key tiles the most queries), so that the blocks that finish
                // last are short.  Without one the run is 1: the tiles of a head, which read the same
                // columns, are neighbours.
                Item it{};
                it.valid = block >= 0;
                if (it.valid) {
                    const int run0 = block / (args.run * args.tiles) * args.run, in_run = block - run0 * args.tiles;
                    const int width = min(args.run, heads * a.seqs - run0), order = in_run / width;
                    const int sh = run0 + in_run - order * width;
                    it.seq = sh / heads;
                    it.head = sh - it.seq * heads;
                    it.r0 = ((MODE == GRAD_KV) == args.ascending ? order : args.tiles - 1 - order) * ROWS;
                    const AttnMask mask(a, it.seq);
                    it.row_len = MODE == GRAD_KV ? mask.k_len : mask.q_len;
                    it.col_len = MODE == GRAD_KV ? mask.q_len : mask.k_len;
                    const int r_last = min(it.r0 + ROWS, it.row_len) - 1;
                    if (r_last >= it.r0) {
                        const int lo = first_col(mask, it.r0), hi = last_col(mask, r_last);
                        if (hi > lo) it.c_begin = lo / COLS, it.per_head = (hi + COLS - 1) / COLS - it.c_begin;
                        it.full_lo = first_col(mask, r_last);
                        it.full_hi = last_col(mask, it.r0);
                    }
                    it.nblk = it.per_head * (MODE == GRAD_KV ? group : 1);
                }
                // (phase k / 2 - 1 of its slot: the next needs this item)
                if (k >= 2) ok = mbar_wait(&item_empty[k & 1], (k / 2 - 1) & 1, err, DEV_TIMEOUT_ATTN_TRAIN);
                if (!ok) break;
                items[k & 1] = it;
                mbar_arrive(&item_full[k & 1]);
                if (!it.valid) break;
                // ---- its loads
                if (it.nblk > 0) {
                    uint64_t* bar = &r_full[n % C::RB];
                    uint8_t* rb = rows + n % C::RB * C::ROW_BYTES;
                    // the buffer's previous item (phase n / RB - 1; the next needs these loads)
                    if (n >= C::RB) ok = mbar_wait(&r_free[n % C::RB], (n / C::RB - 1) & 1, err, DEV_TIMEOUT_ATTN_TRAIN);
                    if (ok) {
                        mbar_arrive_expect_tx(bar, C::ROW_BYTES);
                        // part p of a pair is the maps' sequence p * seqs + seq
#pragma unroll
                        for (int i = 0; i < PARTS * HD / 64; i++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {  // 64 rows each
                                const int o = (2 * i + h) * BOX, d = i % (HD / 64) * 64, sq = i / (HD / 64) * a.seqs + it.seq;
                                tma_load_4d(rb + o, rm1, bar, d, it.r0 + 64 * h, it.head, sq);
                                if (C::GRAD) tma_load_4d(rb + C::RTILE + o, rm2, bar, d, it.r0 + 64 * h, it.head, sq);
                            }
                        n++;
                    }
                    for (int gi = 0; ok && gi < it.nblk; gi++) {
                        const int g = gt + gi;
                        // the stage's previous block (phase g / NST - 1; the one after it needs this load)
                        if (g >= NST) ok = mbar_wait(&c_empty[g % NST], (g / NST - 1) & 1, err, DEV_TIMEOUT_ATTN_TRAIN);
                        if (!ok) {
                            gt = g;
                            break;
                        }
                        uint8_t* st = ring + (g % NST) * C::STAGE;
                        uint64_t* cb = &c_full[g % NST];
                        const int c0 = col0(it, gi), ch = col_head(it, gi);
                        mbar_arrive_expect_tx(cb, 2 * C::CTILE + C::STATS);
#pragma unroll
                        for (int i = 0; i < PARTS * HD / 64; i++) {
                            const int d = i % (HD / 64) * 64, sq = i / (HD / 64) * a.seqs + it.seq;
                            tma_load_4d(st + i * BOX, cm1, cb, d, c0, ch, sq);
                            tma_load_4d(st + C::CTILE + i * BOX, cm2, cb, d, c0, ch, sq);
                        }
                        if (MODE == GRAD_KV)
                            bulk_load(st + 2 * C::CTILE,
                                      args.stats + (((long long)it.seq * a.q_heads + ch) * args.q_tiles * 2 + c0 / COLS) *
                                                       C::STAT_LD,
                                      C::STATS, cb);
                        else if (PAIR)
                            bulk_load(st + 2 * C::CTILE,
                                      args.key_stats + (((long long)it.seq * a.k_heads + ch) * args.k_tiles + c0 / COLS) * kKeyStat,
                                      C::STATS, cb);
                    }
                    if (ok) gt += it.nblk;
                }
                // The next item is claimed once this one's loads are under way, a ring of stages before its end:
                // claimed at its start, the longest items would take the next longest with them.
                // (phase k; the next needs another request)
                mbar_arrive_expect_tx(answered, 16);
                try_cancel(answer, answered);
                const bool came = mbar_wait(answered, k & 1, err, DEV_TIMEOUT_ATTN_TRAIN);
                ok = ok && came;
                block = came ? cancelled_block(answer) : -1;
            }
            // every load has landed before the block may exit (already true unless a wait expired)
            for (int x = max(0, n - C::RB); x < n; x++)
                mbar_wait(&r_full[x % C::RB], (x / C::RB) & 1, err, DEV_TIMEOUT_ATTN_TRAIN);
            for (int x = max(0, gt - NST); x < gt; x++)
                mbar_wait(&c_full[x % NST], (x / NST) & 1, err, DEV_TIMEOUT_ATTN_TRAIN);
        }
    } else if (warp == 1) {
        // ---- T1, T2
        // zeros over rows [from, n) of a tile (boxes of n rows); pairs come with zeros there
        auto clear = [&](uint8_t* tile, int from, int n) {
            for (int i = 0; i < HD / 64; i++)
                for (int x = from * 8 + lane; x < n * 8; x += 32)
                    *reinterpret_cast<uint4*>(tile + i * n * 128 + x * 16) = make_uint4(0, 0, 0, 0);
        };
        const uint32_t t_desc = idesc<T>(COLS, false, false), t_neg = idesc<T>(COLS, false, true);
        bool ok = true;
        Item it;
        for (int k = 0, gt = 0, n = 0; ok && next_uniform(k, it); k++) {
            if (it.nblk == 0) continue;
            uint8_t* rows1 = rows + n % C::RB * C::ROW_BYTES;
            uint8_t* rows2 = rows1 + C::RTILE;
            // (in TMEM phase n, in shared memory phase n / RB; the next needs this item's outputs)
            ok = __all_sync(0xffffffffu,
                            C::ROW_TMEM ? mbar_wait(rows_in, n & 1, err, DEV_TIMEOUT_ATTN_TRAIN)
                                        : mbar_wait(&r_full[n % C::RB], (n / C::RB) & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
            if (!PAIR && !C::ROW_TMEM && ok && it.r0 + ROWS > it.row_len && it.row_len < row_cap) {
                clear(rows1, it.row_len - it.r0, ROWS);
                if (C::GRAD) clear(rows2, it.row_len - it.r0, ROWS);
                fence_async_smem();
                __syncwarp();
            }
            for (int gi = 0; ok && gi < it.nblk; gi++) {
                const int g = gt + gi;
                // The column tiles of block g (phase g / NST; the next needs this block's second product), and the
                // score buffer.  T overwrites the weights of block g - NBUF, which its second products have read
                // (acc_done, phase g / NBUF - 1; the next needs this T).  EARLY: T1 overwrites scores that the softmax
                // has read once its weights are written (p_full, the same phase), and only T2 waits for the products.
                uint64_t* c_bar = &c_full[g % NST];
                uint64_t* t_bar = C::EARLY ? &p_full[g % NBUF] : &acc_done[g % NBUF];
                const uint32_t c_phase = (g / NST) & 1, t_phase = (g / NBUF - 1) & 1;
                ok = __all_sync(0xffffffffu, g >= NBUF ? wait_both(c_bar, c_phase, t_bar, t_phase, err)
                                                       : mbar_wait(c_bar, c_phase, err, DEV_TIMEOUT_ATTN_TRAIN));
                if (!ok) break;
                uint8_t* st = ring + (g % NST) * C::STAGE;
                const int c0 = col0(it, gi);
                if (!PAIR && c0 + COLS > it.col_len && it.col_len < col_cap) {
                    clear(st, it.col_len - c0, COLS);
                    clear(st + C::CTILE, it.col_len - c0, COLS);
                    fence_async_smem();
                    __syncwarp();
                }
                const uint32_t r1 = smem_u32(rows1), r2 = smem_u32(rows2), b = smem_u32(st);
                const uint32_t t = tmem + (g % NBUF) * C::TBUF;
                // T1 (i = 0) or T2.  Pairs: l h + h l + h h, the small products first (the accumulator truncates);
                // the dropped l l is 2^-22 of the product
                auto product = [&](int i) {
#pragma unroll
                    for (int c = 0; c < (PAIR ? 3 : 1); c++)
#pragma unroll
                        for (int kk = 0; kk < HD / 16; kk++) {
                            const uint32_t ro = (i ? r2 : r1) + (PAIR && c == 0 ? RPART : 0) + (kk / 4) * 2 * BOX + (kk % 4) * 32;
                            const uint32_t co = b + i * C::CTILE + (PAIR && c == 1 ? CPART : 0) + (kk / 4) * BOX + (kk % 4) * 32;
                            const uint32_t desc = i == 0 && args.negate ? t_neg : t_desc;
                            if constexpr (C::ROW_TMEM)
                                umma_f16_ts(t + 64 * i, tmem + C::ROWT + i * HD / 2 + kk * 8, desc_k_sw128(co), desc, kk + c != 0);
                            else
                                umma_f16(t + 64 * i, desc_k_sw128(ro), desc_k_sw128(co), desc, kk + c != 0);
                        }
                };
                if (C::EARLY) {
                    tc_fence_after();
                    if (elect_one()) product(0);
                    __syncwarp();
                    if (g >= NBUF)
                        ok = __all_sync(0xffffffffu, mbar_wait(&acc_done[g % NBUF], t_phase, err, DEV_TIMEOUT_ATTN_TRAIN));
                    if (!ok) break;
                }
                tc_fence_after();
                if (elect_one()) {
                    if (!C::EARLY) product(0);
                    if (C::GRAD) product(1);
                    umma_commit(&t_full[g % NBUF]);
                }
                __syncwarp();
            }
            gt += it.nblk;
            n++;
        }
    } else if (warp == 2) {
        // ---- second products: P v (forward); dS k, or dS^T q and P^T dout
        constexpr uint32_t acc_desc = idesc<T>(HD, true);
        // where the weights of columns 16 kk.. are; a pair's h and l, or dkv's dS and P, are side by side
        auto weight_col = [](int kk) { return PAIR || MODE == GRAD_KV ? 16 * kk : 8 * kk; };
        bool ok = true;
        Item it;
        int added[2] = {0, 0};  // pairs: sums of each accumulator taken so far
        for (int k = 0, gt = 0, n = 0; ok && next_uniform(k, it); k++) {
            if (it.nblk == 0) continue;
            // the accumulators of the item before (phase n - 1; the next needs this item's products)
            if (n > 0) ok = __all_sync(0xffffffffu, mbar_wait(acc_read, (n - 1) & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
            for (int gi = 0; ok && gi < it.nblk; gi++) {
                const int g = gt + gi;
                // the column tiles (as above) and the weights of block g (phase g / NBUF; the next needs T of
                // block g + NBUF, hence this product)
                ok = __all_sync(0xffffffffu, wait_both(&c_full[g % NST], (g / NST) & 1, &p_full[g % NBUF], (g / NBUF) & 1, err));
                // which accumulator, and the block's number there: a pair's starts afresh every second one,
                // once the softmax group has added it up (the next addition needs this product)
                const int which = MODE == FORWARD ? g % NWG : 0, m = MODE == FORWARD ? gi / NWG : gi;
                if (C::SUM && ok && m >= 2 && m % 2 == 0) {
                    ok = __all_sync(0xffffffffu,
                                    mbar_wait(&acc_free[which], added[which] & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
                    added[which]++;
                }
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t b = smem_u32(ring + (g % NST) * C::STAGE);
                    const uint32_t t = tmem + (g % NBUF) * C::TBUF;
                    const uint32_t acc = tmem + C::ACC + which * HD;
                    const uint32_t first = C::SUM ? m % 2 == 0 : m == 0;
                    auto second = [&](uint32_t d, uint32_t weights, uint32_t tile) {
#pragma unroll
                        for (int c = 0; c < (PAIR ? 3 : 1); c++)
#pragma unroll
                            for (int kk = 0; kk < COLS / 16; kk++)
                                umma_f16_ts(d, weights + weight_col(kk) + (PAIR && c == 0 ? 8 : 0),
                                            desc_mn_sw128(tile + (PAIR && c == 1 ? CPART : 0) + kk * 2048), acc_desc,
                                            kk + c != 0 || !first);
                    };
                    second(acc, t + (C::GRAD ? 64 : 0), b + (MODE == FORWARD ? C::CTILE : 0));
                    if (MODE == GRAD_KV) second(acc + HD, PAIR ? t : t + 64 + 8, b + C::CTILE);
                    umma_commit(&acc_done[g % NBUF]);
                    umma_commit(&c_empty[g % NST]);
                    if (gi == it.nblk - 1) umma_commit(all_done);
                }
                __syncwarp();
            }
            gt += it.nblk;
            n++;
        }
    } else {
        // ---- softmax: TMEM lane quadrant warp % 4, one row per thread
        const int wg = (warp - C::SOFTMAX) / 4;
        const int qd = warp & 3, r = qd * 32 + lane;
        const uint32_t lb = tmem + (static_cast<uint32_t>(qd * 32) << 16);
        // (pairs: the scores are in units of log2 once they are read)
        const float k2 = PAIR ? 1.0f : args.k2;
        constexpr float P_LOG2 = !F16 || PAIR ? 0.0f : MODE == FORWARD ? 7.0f : MODE == GRAD_KV ? 10.0f : 0.0f;
        constexpr float P_SCALE = 1024.0f;  // 2^P_LOG2 of dkv
        int pairs = 0;  // pairs, gradients: pairs of blocks of the items before
        bool ok = true;
        Item it;
        for (int k = 0, gt = 0, n = 0; next_item(k, it); k++) {
            const int seq = it.seq, head = it.head, r0 = it.r0, row = r0 + r, nblk = it.nblk;
            const bool live = row < it.row_len;
            const AttnMask mask(a, it.seq, it.row_len, it.col_len, MODE == GRAD_KV);
            const int lo = first_col(mask, row), hi = last_col(mask, row);
            float* join = joins + (k & 1) * C::JOIN;
            uint8_t* rows1 = rows + n % C::RB * C::ROW_BYTES;  // the staging of the outputs, at the end
            // this row in a fp32 output
            auto out_row = [&](const HeadsView& t) {
                return static_cast<float*>(t.p) + (long long)seq * t.seq + (long long)head * t.head + (long long)row * t.row;
            };

            // The row tiles go to TMEM as the A operands of T; what they held for the item before was read by
            // products that its all_done covers.  Rows past the length are zeros there.
            if (C::ROW_TMEM && nblk > 0) {
                // (phase n / RB; the next needs this item's outputs)
                ok = __all_sync(0xffffffffu, ok && mbar_wait(&r_full[n % C::RB], (n / C::RB) & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
#pragma unroll 1
                for (int i = wg; i < (C::GRAD ? 2 : 1) * HD / 64; i += NWG) {  // 64 elements: 32 columns
                    const uint8_t* from = rows1 + i * 2 * BOX + r * 128;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint4 x = *reinterpret_cast<const uint4*>(from + (((4 * h + j) ^ (r & 7)) << 4));
                            w[4 * j] = live ? x.x : 0, w[4 * j + 1] = live ? x.y : 0;
                            w[4 * j + 2] = live ? x.z : 0, w[4 * j + 3] = live ? x.w : 0;
                        }
                        tmem_st16(lb + C::ROWT + i * 32 + h * 16, w);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(rows_in);
            }

            // dq, 16-bit: does the row see keys of one block only?  Then D is taken from that block (below)
            const bool single = MODE == GRAD_Q && !PAIR && live && hi > lo && (hi - 1) / COLS == lo / COLS;
            // dq: this row's -lse log2 e, -D and fp16 scale; dkv: the fp16 scale of the head group
            float nlse = 0.0f, ndot = 0.0f, ds_scale = 1.0f;
            // pairs: this row's factors of T1 and T2
            float row1 = 0.0f, row2 = 0.0f;
            if (PAIR && MODE == GRAD_KV) {
                const float* st =
                    args.key_stats + (((long long)seq * a.k_heads + head) * args.k_tiles + row / 64) * kKeyStat + row % 64;
                if (live) row1 = args.k2 * st[0], row2 = st[64];
            } else if (PAIR) {
                const float* st =
                    args.stats + ((((long long)seq * a.q_heads + head) * args.q_tiles + r0 / ROWS) * 2 + r / 64) * C::STAT_LD + r % 64;
                if (live) row1 = args.k2 * st[128];
                if (MODE == GRAD_Q) {
                    nlse = live ? st[0] : -INFINITY;
                    ndot = live ? st[64] : 0.0f;
                    row2 = live ? st[192] : 0.0f;
                }
            } else if (MODE == GRAD_Q) {
                const long long sqh = (long long)seq * a.q_heads + head;
                float norm2 = 0.0f;
                nlse = -INFINITY;
                if (live) {
                    const T* o = static_cast<const T*>(a.o.p) + seq * a.o.seq + head * a.o.head + (long long)row * a.o.row;
                    const T* d =
                        static_cast<const T*>(a.dout.p) + seq * a.dout.seq + head * a.dout.head + (long long)row * a.dout.row;
                    float dot = 0.0f;
#pragma unroll 4
                    for (int c = 0; c < HD; c += 8) {
                        Vec<T, 8> vo, vd;
                        vo.load(o + c);
                        vd.load(d + c);
                        float x[8], y[8];
                        vo.get(x);
                        vd.get(y);
#pragma unroll
                        for (int i = 0; i < 8; i++) dot += x[i] * y[i], norm2 += y[i] * y[i];
                    }
                    ndot = -dot;
                    const float l = a.lse[sqh * a.q_rows + row];
                    if (l != -INFINITY) nlse = row_nlse(l);
                }
                const float norm = sqrtf(norm2);
                if (F16) ds_scale = 8.0f * inverse_power(norm);
                if (wg == 0) {
                    float* st = args.stats + ((sqh * args.q_tiles + r0 / ROWS) * 2 + r / 64) * 128 + r % 64;
                    st[0] = nlse;
                    if (!single) st[64] = ndot;
                    if (F16) {
                        float m = norm;
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        if (lane == 0) join[qd] = m;
                        asm volatile("bar.sync 1, 128;" ::: "memory");
                        if (r == 0)
                            args.norms[sqh * args.q_tiles + r0 / ROWS] = fmaxf(fmaxf(join[0], join[1]), fmaxf(join[2], join[3]));
                    }
                }
            }
            if (MODE == GRAD_KV && F16 && !PAIR) {
                // the largest |dout row| of the head group, from one for each tile
                float m = 0.0f;
                const float* n = args.norms + ((long long)seq * a.q_heads + head * group) * args.q_tiles;
                for (int i = lane; i < group * args.q_tiles; i += 32) m = fmaxf(m, n[i]);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                ds_scale = 8.0f * inverse_power(m);
            }

            float m = -INFINITY, l = 0.0f;  // forward: running maximum (raw scores) and sum (times 2^P_LOG2)
            float m_sum = -INFINITY;        // pairs, forward: the maximum that the summed accumulators refer to
            auto sum_factor = [&](float to) { return m_sum == to ? 1.0f : ex2_approx((m_sum - to) * k2); };
            // pairs: the units of this row's weights (dkv: of dS and of P) in the accumulators; 0: all were 0 so far
            float unit1 = 0.0f, unit2 = 0.0f;
            // the unit after a block whose largest weight is `top`: a first block (of two) takes its own, a second one the
            // first one's if its weights fit there.  Returns what the accumulator is to be multiplied by.
            auto new_unit = [&](float& unit, float top, bool first) {
                const float before = unit;
                if (first || before == 0.0f) {
                    unit = top > 0.0f ? weight_unit(top) : 0.0f;
                    return 1.0f;
                }
                if (!(top * before > MAX_WEIGHT)) return 1.0f;
                unit = weight_unit(top);
                return unit / before;
            };
            auto used = [](float unit) { return unit == 0.0f ? 1.0f : unit; };
            // multiplies `n` columns of an accumulator of this warp's rows
            auto scale_acc = [&](uint32_t acc, int n, float by) {
                const uint64_t c2 = pack2(by, by);
#pragma unroll 1
                for (int cb = 0; cb < n; cb += 16) {
                    float o[16];
                    uint32_t u[16];
                    tmem_ld16(acc + cb, o);
#pragma unroll
                    for (int d = 0; d < 16; d += 2) {
                        unpack2(mul2(pack2(o[d], o[d + 1]), c2), o[d], o[d + 1]);
                        u[d] = __float_as_uint(o[d]), u[d + 1] = __float_as_uint(o[d + 1]);
                    }
                    tmem_st16(acc + cb, u);
                }
            };
            for (int gi = NWG == 1 ? 0 : (wg + gt) & 1; gi < nblk; gi += NWG) {
                const int g = gt + gi, buf = g % NBUF, c0 = col0(it, gi);
                const uint32_t t = lb + buf * C::TBUF;
                const bool full = c0 >= it.full_lo && c0 + COLS <= it.full_hi;
                // T of block g (phase g / NBUF of its buffer: the next needs this block's weights).  After an
                // expired wait the loop keeps running (results unused).
                // Column statistics came by bulk copy: this thread's own wait makes them visible.
                uint64_t *t_bar = &t_full[buf], *c_bar = &c_full[g % NST];
                ok = __all_sync(0xffffffffu, ok && (C::STATS > 0 ? wait_both(t_bar, (g / NBUF) & 1, c_bar, (g / NST) & 1, err)
                                                                 : mbar_wait(t_bar, (g / NBUF) & 1, err, DEV_TIMEOUT_ATTN_TRAIN)));
                tc_fence_after();
                const int nth = MODE == FORWARD ? gi / NWG : gi;  // the block's number in its accumulator
                const float4* st = reinterpret_cast<const float4*>(ring + (g % NST) * C::STAGE + 2 * C::CTILE);
                if constexpr (MODE == FORWARD) {
                    float s[64];
                    tmem_ld32(t, s);
                    tmem_ld32(t + 32, s + 32);
                    // Pairs: the units of the columns; the row's factor, which may be 0, before -inf takes a score's place
                    const float kf = !PAIR ? args.k2 : full ? row1 : 1.0f;
                    if constexpr (PAIR) {
#pragma unroll
                        for (int c = 0; c < 64; c += 4) {
                            const float4 kk = lds4(st + c / 4);
                            unpack2(mul2(pack2(s[c], s[c + 1]), pack2(kk.x, kk.y)), s[c], s[c + 1]);
                            unpack2(mul2(pack2(s[c + 2], s[c + 3]), pack2(kk.z, kk.w)), s[c + 2], s[c + 3]);
                        }
                    }
                    if (!full) {
#pragma unroll
                        for (int c = 0; c < 64; c++) {
                            if (PAIR) s[c] *= row1;
                            if (c0 + c < lo || c0 + c >= hi) s[c] = -INFINITY;
                        }
                    }
                    float mx[8];
#pragma unroll
                    for (int c = 0; c < 8; c++) mx[c] = fmaxf(s[c], s[c + 8]);
#pragma unroll
                    for (int c = 16; c < 64; c += 16)
#pragma unroll
                        for (int i = 0; i < 8; i++) mx[i] = max3f(mx[i], s[c + i], s[c + 8 + i]);
                    const float mb = max3f(max3f(mx[0], mx[1], mx[2]), max3f(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) *
                                     (PAIR ? kf : 1.0f);
                    // (an unseen block leaves mb = -inf: no raise, and the exponents below stay -inf)
                    const bool raise = mb > m && (mb - m) * k2 > RESCALE_LOG2;
                    const float corr = raise ? ex2_approx((m - mb) * k2) : 1.0f;  // 0 from m = -inf
                    if (raise) m = mb;
                    float off = m == -INFINITY ? 0.0f : P_LOG2 - m * k2, ks = kf;
                    // Huge scores: off is rounded by up to 2^-24 of it, by which every weight of the row would be off: in
                    // fp16 they would pass 2^16, or vanish.  There the maximum is subtracted first.  (bf16 holds any such
                    // factor and the row sum takes it out again; the test alone cost 2 % of 128 windows of 384 rows.)
                    if ((F16 || PAIR) && fabsf(off) > FAR) {
#pragma unroll
                        for (int c = 0; c < 64; c++) s[c] = PAIR ? __fmul_rn(s[c], kf) - m : s[c] - m;
                        off = P_LOG2;
                        if (PAIR) ks = 1.0f;
                    }
                    const uint64_t k22 = pack2(ks, ks), off2 = pack2(off, off);
                    uint64_t sum2[4] = {0, 0, 0, 0};
                    float acc_by = corr;  // what the accumulator is multiplied by
                    if constexpr (PAIR) {
                        float top = 0.0f, tops[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int c = 0; c < 64; c += 4) {
                            const float4 vv = lds4(st + 16 + c / 4);
#pragma unroll
                            for (int e = c; e < c + 4; e += 2) {
                                float x, y;
                                unpack2(fma2(pack2(s[e], s[e + 1]), k22, off2), x, y);
                                const uint64_t p2 = pack2(ex2_approx(x), ex2_approx(y));
                                sum2[(e >> 1) & 3] = add2(sum2[(e >> 1) & 3], p2);
                                unpack2(mul2(p2, e == c ? pack2(vv.x, vv.y) : pack2(vv.z, vv.w)), s[e], s[e + 1]);
                                tops[(e >> 1) & 3] = max3f(tops[(e >> 1) & 3], s[e], s[e + 1]);
                            }
                        }
                        top = fmaxf(max3f(tops[0], tops[1], tops[2]), tops[3]);
                        acc_by *= new_unit(unit1, top, nth % 2 == 0);
                        const float by = used(unit1);
#pragma unroll
                        for (int i = 0; i < 64; i += 16) {  // 8 words of h and 8 of l
                            uint32_t w[16];
#pragma unroll
                            for (int c = 0; c < 16; c += 2) split2x2(s[i + c], s[i + c + 1], by, w[c / 2], w[8 + c / 2]);
                            tmem_st16(t + i, w);
                        }
                    } else {
                        // 16 words of weights at a time, over scores that are in registers
#pragma unroll
                        for (int i = 0; i < 64; i += 32) {
                            uint32_t w[16];
#pragma unroll
                            for (int c = i; c < i + 32; c += 2) {
                                float x, y;
                                unpack2(fma2(pack2(s[c], s[c + 1]), k22, off2), x, y);
                                x = ex2_approx(x);
                                y = ex2_approx(y);
                                sum2[(c >> 1) & 3] = add2(sum2[(c >> 1) & 3], pack2(x, y));
                                w[(c - i) / 2] = pack_pair<T>(x, y);
                            }
                            tmem_st16(t + i / 2, w);
                        }
                    }
                    float sa, sb;
                    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), sa, sb);
                    l = l * corr + (sa + sb);
                    if (nth > 0 && !(C::SUM && nth % 2 == 0) && __any_sync(0xffffffffu, acc_by != 1.0f)) {
                        // this group's previous product (its phase: the buffer's next product needs P of
                        // this or a later block of the group)
                        ok = __all_sync(0xffffffffu, ok && mbar_wait(&acc_done[(g - NWG) % NBUF], ((g - NWG) / NBUF) & 1, err,
                                                                     DEV_TIMEOUT_ATTN_TRAIN));
                        tc_fence_after();
                        scale_acc(lb + C::ACC + wg * HD, HD, acc_by);
                    }
                } else {
                    const uint64_t k22 = pack2(k2, k2), scale2 = pack2(ds_scale, ds_scale);
                    // A row of few keys has large P, and dP - D cancels: with D from the rounded output, dS would
                    // keep that rounding (a row with one key has dS = 0).  Where the row's keys are all here,
                    // D = sum P dP, for dkv too.
                    if constexpr (MODE == GRAD_Q && !PAIR) {
                        const bool here = single && lo / COLS * COLS == c0;
                        if (__any_sync(0xffffffffu, here)) {
                            float d = 0.0f;
#pragma unroll 1
                            for (int h = 0; h < COLS; h += 16) {
                                float s[16], u[16];
                                tmem_ld_pair(t + h, t + 64 + h, s, u);
#pragma unroll
                                for (int c = 0; c < 16; c++) {
                                    const int cc = c0 + h + c;
                                    if (cc >= lo && cc < hi) d += ex2_approx(fmaf(s[c], k2, nlse)) * u[c];
                                }
                            }
                            if (here) {
                                ndot = -d;
                                args.stats[((((long long)seq * a.q_heads + head) * args.q_tiles + r0 / ROWS) * 2 + r / 64) * 128 +
                                           64 + r % 64] = ndot;
                            }
                        }
                    }
                    auto weights = [&](auto masked) {
                        constexpr int CH = 16;  // columns in registers at a time
                        // dkv: the statistics (-lse log2 e, -D) that are read before the wait for the scores, as many
                        // as registers hold.  2 x 4096 rows, 16 heads of 128: gradient 904 us with both, 914 with none;
                        // of 64 with both 677, with one 682, with none 700, but both spill there and fp16 takes
                        // 154 us for 64 windows of 384 rows, 151 with one or none.
                        constexpr int AHEAD = MODE != GRAD_KV ? 0 : C::SMALL ? 1 : 2;
#pragma unroll
                        for (int h = 0; h < COLS; h += CH) {  // the weights go over scores that are read already
                            float s[CH], u[CH];
                            float4 sl[CH / 4], sd[CH / 4];
#pragma unroll
                            for (int c = 0; c < CH / 4; c++) {
                                if (AHEAD > 0) sl[c] = st[h / 4 + c];
                                if (AHEAD > 1) sd[c] = st[16 + h / 4 + c];
                            }
                            tmem_ld_pair(t + h, t + 64 + h, s, u);
                            uint32_t w[CH], *dw = w, *pw = w + CH / 2;
#pragma unroll
                            for (int c = 0; c < CH; c += 4) {
                                float4 nl = make_float4(nlse, nlse, nlse, nlse), nd = make_float4(ndot, ndot, ndot, ndot);
                                if (MODE == GRAD_KV) {
                                    nl = AHEAD > 0 ? sl[c / 4] : st[(h + c) / 4];
                                    nd = AHEAD > 1 ? sd[c / 4] : st[16 + (h + c) / 4];
                                }
#pragma unroll
                                for (int e = 0; e < 4; e += 2) {
                                    const uint64_t n2 = e == 0 ? pack2(nl.x, nl.y) : pack2(nl.z, nl.w);
                                    const uint64_t d2 = e == 0 ? pack2(nd.x, nd.y) : pack2(nd.z, nd.w);
                                    const int cc = c0 + h + c + e;
                                    float x, y, gx, gy;
                                    unpack2(fma2(pack2(s[c + e], s[c + e + 1]), k22, n2), x, y);
                                    x = ex2_approx(x);
                                    y = ex2_approx(y);
                                    if (masked && (cc < lo || cc >= hi)) x = 0.0f;
                                    if (masked && (cc + 1 < lo || cc + 1 >= hi)) y = 0.0f;
                                    uint64_t g2 = mul2(pack2(x, y), add2(pack2(u[c + e], u[c + e + 1]), d2));
                                    if (F16) g2 = mul2(g2, scale2);
                                    unpack2(g2, gx, gy);
                                    if (masked && x == 0.0f) gx = 0.0f;
                                    if (masked && y == 0.0f) gy = 0.0f;
                                    const int i = (c + e) / 2;
                                    if (MODE == GRAD_KV)
                                        pw[i] = F16 ? pack_pair<T>(x * P_SCALE, y * P_SCALE) : pack_pair<T>(x, y);
                                    dw[i] = pack_pair<T>(gx, gy);
                                }
                            }
                            if constexpr (MODE == GRAD_KV)
                                tmem_st16(t + 64 + h, w);  // both over T2
                            else
                                tmem_st8(t + 64 + h / 2, dw);
                        }
                    };
                    // Pairs: dS (and P) times the units of their columns, first as they are, for their largest, then
                    // in the row's unit as h and l; meanwhile they are in TMEM, over T2 and over the scores.
                    auto pair_weights = [&](auto masked) {
                        constexpr int CH = 16;
                        constexpr bool KV = MODE == GRAD_KV;
                        const uint64_t row12 = pack2(row1, row1), row22 = pack2(row2, row2);
                        float top1 = 0.0f, top2 = 0.0f;
#pragma unroll
                        for (int h = 0; h < COLS; h += CH) {
                            float s[CH], u[CH];
                            tmem_ld_pair(t + h, t + 64 + h, s, u);
#pragma unroll
                            for (int c = 0; c < CH; c += 4) {
                                // units of the columns of T1 and T2 (k and v, or q and dout)
                                const float4 a4 = lds4(st + (KV ? 32 : 0) + (h + c) / 4), b4 = lds4(st + (KV ? 48 : 16) + (h + c) / 4);
                                float4 nl = make_float4(nlse, nlse, nlse, nlse), nd = make_float4(ndot, ndot, ndot, ndot);
                                if (KV) nl = lds4(st + (h + c) / 4), nd = lds4(st + 16 + (h + c) / 4);
#pragma unroll
                                for (int e = 0; e < 4; e += 2) {
                                    const uint64_t n2 = e == 0 ? pack2(nl.x, nl.y) : pack2(nl.z, nl.w);
                                    const uint64_t d2 = e == 0 ? pack2(nd.x, nd.y) : pack2(nd.z, nd.w);
                                    const uint64_t a2 = e == 0 ? pack2(a4.x, a4.y) : pack2(a4.z, a4.w);
                                    const uint64_t b2 = e == 0 ? pack2(b4.x, b4.y) : pack2(b4.z, b4.w);
                                    const int i = c + e, cc = c0 + h + i;
                                    float x, y, gx, gy;
                                    unpack2(fma2(mul2(pack2(s[i], s[i + 1]), a2), row12, n2), x, y);
                                    x = ex2_approx(fminf(x, 0.0f));  // (row_nlse: huge scores)
                                    y = ex2_approx(fminf(y, 0.0f));
                                    if (masked && (cc < lo || cc >= hi)) x = 0.0f;
                                    if (masked && (cc + 1 < lo || cc + 1 >= hi)) y = 0.0f;
                                    const uint64_t g2 = mul2(pack2(x, y), fma2(mul2(pack2(u[i], u[i + 1]), b2), row22, d2));
                                    unpack2(mul2(g2, a2), gx, gy);
                                    if (masked && x == 0.0f) gx = 0.0f;
                                    if (masked && y == 0.0f) gy = 0.0f;
                                    if (KV) unpack2(mul2(pack2(x, y), b2), s[i], s[i + 1]);
                                    u[i] = gx, u[i + 1] = gy;
                                }
                            }
                            uint32_t w[CH];
                            if (KV) {
                                top2 = max16(s, top2);
#pragma unroll
                                for (int c = 0; c < CH; c++) w[c] = __float_as_uint(s[c]);
                                tmem_st16(t + h, w);
                            }
                            top1 = max16(u, top1);
#pragma unroll
                            for (int c = 0; c < CH; c++) w[c] = __float_as_uint(u[c]);
                            tmem_st16(t + 64 + h, w);
                        }
                        // The row's units: an even block's go to the group of the next one, which goes on with them.
                        // (unit_set: phase x / 2 of its slot for pair x.  The slot is set again two pairs on, by a block at least
                        // four on; its T2 waits for the products of a block three before it or two, hence for this pair's
                        // second one's weights.)
                        const int x = pairs + gi / 2;
                        float* const xu = units + (x & 1) * 256;
                        float by1 = 1.0f, by2 = 1.0f;
                        if (gi % 2 == 0) {
                            new_unit(unit1, top1, true);
                            if (KV) new_unit(unit2, top2, true);
                            if (gi + 1 < nblk) {
                                xu[r] = unit1;
                                if (KV) xu[128 + r] = unit2;
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&unit_set[x & 1]);
                            }
                        } else {
                            ok = __all_sync(0xffffffffu, ok && mbar_wait(&unit_set[x & 1], (x >> 1) & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
                            unit1 = xu[r];
                            by1 = new_unit(unit1, top1, false);
                            if (KV) unit2 = xu[128 + r], by2 = new_unit(unit2, top2, false);
                            if (__any_sync(0xffffffffu, by1 != 1.0f || by2 != 1.0f)) {
                                // the even block's product (its phase: the next product of its buffer follows this block's)
                                ok = __all_sync(0xffffffffu, ok && mbar_wait(&acc_done[(g - 1) % NBUF], ((g - 1) / NBUF) & 1, err,
                                                                             DEV_TIMEOUT_ATTN_TRAIN));
                                tc_fence_after();
                                scale_acc(lb + C::ACC, HD, by1);
                                if (KV) scale_acc(lb + C::ACC + HD, HD, by2);
                            }
                        }
                        const float u1 = used(unit1), u2 = used(unit2);
                        tmem_wait_st();  // what is read again
#pragma unroll
                        for (int h = 0; h < COLS; h += CH) {
                            float d[CH];
                            uint32_t w[CH];
                            if constexpr (KV) {
                                float p[CH];
                                tmem_ld_pair(t + h, t + 64 + h, p, d);
#pragma unroll
                                for (int c = 0; c < CH; c += 2) split2x2(p[c], p[c + 1], u2, w[c / 2], w[8 + c / 2]);
                                tmem_st16(t + h, w);
                            } else {
                                tmem_ld16(t + 64 + h, d);
                            }
#pragma unroll
                            for (int c = 0; c < CH; c += 2) split2x2(d[c], d[c + 1], u1, w[c / 2], w[8 + c / 2]);
                            tmem_st16(t + 64 + h, w);
                        }
                    };
                    if constexpr (PAIR)
                        full ? pair_weights(std::false_type()) : pair_weights(std::true_type());
                    else
                        full ? weights(std::false_type()) : weights(std::true_type());
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[buf]);

                // pairs: after every second product into an accumulator, if another follows, add it to the sum
                if (C::SUM && nth % 2 == 1 && gi + (MODE == FORWARD ? NWG : 1) < nblk) {
                    // (its phase: the buffer's next product needs weights of this group)
                    ok = __all_sync(0xffffffffu,
                                    ok && mbar_wait(&acc_done[buf], (g / NBUF) & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
                    tc_fence_after();
                    const float f = MODE == FORWARD ? sum_factor(m) : 1.0f;
                    const float to1 = 1.0f / used(unit1), to2 = 1.0f / used(unit2);  // exact
                    const uint32_t from = lb + C::ACC + (MODE == FORWARD ? wg * HD : 0);
                    constexpr int WIDTH = MODE == GRAD_KV ? 2 * HD : HD;
#pragma unroll 1
                    for (int cb = 0; cb < WIDTH; cb += 16) {
                        float o[16], u[16];
                        tmem_ld16(from + cb, o);
#pragma unroll
                        for (int d = 0; d < 16; d++) o[d] *= cb < HD ? to1 : to2;
                        if constexpr (C::SUM_OUT) {
                            if (live) {
                                float* to = out_row(cb < HD ? a.dk : a.dv) + cb % HD;
#pragma unroll
                                for (int d = 0; d < 16; d++) to[d] = nth == 1 ? o[d] : to[d] + o[d];
                            }
                        } else {
                            if (nth > 1) tmem_ld16(from + C::NACC * HD + cb, u);
                            uint32_t w[16];
#pragma unroll
                            for (int d = 0; d < 16; d++) w[d] = __float_as_uint(nth > 1 ? u[d] * f + o[d] : o[d]);
                            tmem_st16(from + C::NACC * HD + cb, w);
                        }
                    }
                    m_sum = m;
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_free[MODE == FORWARD ? wg : 0]);
                }
            }

            if (nblk == 0) {
                // nothing is seen: zeros, straight to the outputs
                if (MODE == FORWARD && a.lse && wg == 0 && row < a.q_rows)
                    a.lse[((long long)seq * a.q_heads + head) * a.q_rows + row] = -INFINITY;
                for (int o = 0; o < (MODE == GRAD_KV ? 2 : 1); o++) {
                    const HeadsView& t = MODE == FORWARD ? a.o : MODE == GRAD_Q ? a.dq : o ? a.dv : a.dk;
                    using Out = typename std::conditional<PAIR, float, T>::type;
                    Out* p = static_cast<Out*>(t.p) + (long long)seq * t.seq + (long long)head * t.head;
                    // 16-bit rows are whole 16-byte words, fp32 rows may start anywhere
                    constexpr int N = PAIR ? 1 : 8, PER_ROW = HD / N;
                    for (int i = threadIdx.x - 32 * C::SOFTMAX; i < ROWS * PER_ROW; i += 128 * NWG) {
                        const int rr = r0 + i / PER_ROW;
                        if (rr >= row_cap) break;
                        Out* to = p + (long long)rr * t.row + i % PER_ROW * N;
                        if constexpr (PAIR)
                            *to = 0.0f;
                        else
                            *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
                    }
                }
                continue;
            }
            // ---- the accumulators, once every product has completed (phase n; the next needs acc_read)
            ok = __all_sync(0xffffffffu, ok && mbar_wait(all_done, n & 1, err, DEV_TIMEOUT_ATTN_TRAIN));
            tc_fence_after();
            if (PAIR && MODE != FORWARD) {
                // the last block's group knows the accumulators' units (and SUM_OUT: the sums in the outputs are written)
                if (((wg + gt + nblk - 1) & 1) == 0) {
                    join[r] = 1.0f / used(unit1);
                    join[128 + r] = 1.0f / used(unit2);
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                pairs += nblk / 2;
            }
            float f0 = 0.0f, f1 = 0.0f, fv = 1.0f;  // what the accumulator(s) are multiplied by
            float g0 = 0.0f, g1 = 0.0f;  // and their sums
            if (MODE == FORWARD) {
                float lse;
                if (NWG == 1) {
                    g0 = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : NAN;
                    f0 = g0 / used(unit1);
                    g0 *= sum_factor(m);
                    lse = row_lse(l, m, k2, P_LOG2);
                } else {
                    // Joined by the groups' parts in the item, not their numbers: the group of the first block depends on
                    // the items this block of threads had before, and the join is not symmetric in its roundings.
                    const int part = (wg + gt) & 1;
                    join[part * 128 + r] = m;
                    join[256 + part * 128 + r] = l;
                    if (C::SUM) join[512 + part * 128 + r] = sum_factor(m), join[768 + part * 128 + r] = 1.0f / used(unit1);
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                    const float m0 = join[r], m1 = join[128 + r], l0 = join[256 + r], l1 = join[256 + 128 + r];
                    const float mm = fmaxf(m0, m1);
                    // (what saw nothing has m = -inf and l = 0)
                    const float e0 = l0 == 0.0f ? 0.0f : ex2_approx((m0 - mm) * k2);
                    const float e1 = l1 == 0.0f ? 0.0f : ex2_approx((m1 - mm) * k2);
                    const float sum = l0 * e0 + l1 * e1;
                    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : NAN;
                    f0 = e0 * inv;
                    f1 = e1 * inv;
                    lse = row_lse(sum, mm, k2, P_LOG2);
                }
                if (a.lse && wg == 0 && row < a.q_rows)
                    a.lse[((long long)seq * a.q_heads + head) * a.q_rows + row] = live ? lse : -INFINITY;
                if (C::SUM && NWG > 1) {
                    g0 = f0 * join[512 + r];
                    g1 = f1 * join[512 + 128 + r];
                    f0 *= join[768 + r];
                    f1 *= join[768 + 128 + r];
                }
            } else if (PAIR) {
                g0 = args.factor;
                f0 = g0 * join[r];
                fv = join[128 + r];  // of dv
            } else {
                f0 = args.factor / ds_scale;
                if (F16) fv = 1.0f / P_SCALE;
            }
            // 64 columns of an accumulator (plus what belongs to it) to this row's staging: a row of 64
            // elements, its 16-byte words swizzled by the row
            constexpr int EL = PAIR ? 4 : 2, WORDS = 64 * EL / 16, ROW = 64 * EL;
            // (second: the other group's accumulator; summed: what was added up before)
            // The groups of the forward pass take turns, from the group of block gt, whose accumulator comes first.
            constexpr bool TURNS = MODE == FORWARD && NWG > 1;
            const int lead = TURNS ? (gt & 1) * HD : 0;
            const bool second = TURNS && nblk > 1;
            const bool summed = C::SUM && (TURNS ? nblk > 4 : nblk > 2), summed2 = C::SUM && TURNS && nblk > 5;
            auto stage_box = [&](uint32_t col, float f, float gs, const float* sum_row, uint8_t* box) {
                const uint32_t acc = col + lead, acc2 = col + HD - lead;
                const uint32_t sum = acc + C::NACC * HD, sum2 = acc2 + C::NACC * HD;
#pragma unroll 1
                for (int cb = 0; cb < 64; cb += 16) {
                    float o[16], o2[16], u[16], u2[16];
                    tmem_ld16(acc + cb, o);
                    if (second) tmem_ld16(acc2 + cb, o2);
                    if (C::SUM_OUT) {
#pragma unroll
                        for (int d = 0; d < 16; d++) u[d] = summed && live ? sum_row[cb + d] : 0.0f;
                    } else if (summed) {
                        tmem_ld16(sum + cb, u);
                    }
                    if (summed2) tmem_ld16(sum2 + cb, u2);
                    uint32_t w[4 * EL];
#pragma unroll
                    for (int d = 0; d < 16; d += 2) {
                        float x = 0.0f, y = 0.0f;
                        if (live) {
                            x = o[d] * f, y = o[d + 1] * f;
                            if (summed) x += u[d] * gs, y += u[d + 1] * gs;
                            if (second) x += o2[d] * f1, y += o2[d + 1] * f1;
                            if (summed2) x += u2[d] * g1, y += u2[d + 1] * g1;
                        }
                        if constexpr (PAIR)
                            w[d] = __float_as_uint(x), w[d + 1] = __float_as_uint(y);
                        else
                            w[d / 2] = pack_pair<T>(x, y);
                    }
#pragma unroll
                    for (int i = 0; i < EL; i++)
                        *reinterpret_cast<uint4*>(box + r * ROW + (((cb * EL / 16 + i) ^ (r & (WORDS - 1))) << 4)) =
                            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
            };
            // a warp's 32 rows of the staging: one TMA store of 16-bit rows; fp32 rows, whose tensors may have
            // any strides, two rows at a time
            auto send_box = [&](const CUtensorMap* map, const HeadsView& t, uint8_t* box, int d) {
                const int first = r0 + qd * 32;
                if constexpr (PAIR) {
                    __syncwarp();
                    const int word = lane % 16;
                    float* p = static_cast<float*>(t.p) + (long long)seq * t.seq + (long long)head * t.head + d + 4 * word;
                    const bool wide = ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(t.row * 4)) & 15) == 0;
                    for (int i = lane / 16; i < 32 && first + i < row_cap; i += 2) {
                        const int rr = qd * 32 + i;
                        const float4 v = *reinterpret_cast<const float4*>(box + rr * ROW + ((word ^ (rr & 15)) << 4));
                        float* to = p + (long long)(first + i) * t.row;
                        if (wide)
                            *reinterpret_cast<float4*>(to) = v;
                        else
                            to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
                    }
                } else {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0 && first < row_cap) {
                        tma_store_4d(map, box + qd * 32 * ROW, d, first, head, seq);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            };
            // the row tiles are no longer read: they hold the staging, a box of 128 rows for every 64 columns
            const uint32_t acc = lb + C::ACC;
            constexpr int PER = HD / 64, BOXES = MODE == GRAD_KV ? 2 * PER : PER;  // out, dq, or dk then dv
            static_assert(BOXES * ROWS * ROW <= C::ROW_BYTES, "the staging fits the row tiles");
#pragma unroll 1
            for (int i = wg; i < BOXES; i += NWG) {
                uint8_t* box = rows1 + i * ROWS * ROW;
                const int d = 64 * (i % PER);
                const bool is_dv = MODE == GRAD_KV && i >= PER;
                stage_box(acc + 64 * i, is_dv ? fv : f0, is_dv ? 1.0f : g0,
                          C::SUM_OUT ? out_row(is_dv ? a.dv : a.dk) + d : nullptr, box);
                send_box(MODE == FORWARD ? &maps.out : MODE == GRAD_Q ? &maps.dq : i < PER ? &maps.dk : &maps.dv,
                         MODE == FORWARD ? a.o : MODE == GRAD_Q ? a.dq : i < PER ? a.dk : a.dv, box, d);
            }
            // ---- the accumulators are read, and (once the stores have read it) the staging, which the next loads
            // overwrite
            tc_fence_before();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(acc_read);
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                mbar_arrive(&r_free[n % C::RB]);
            }
            gt += nblk;
            n++;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
}

template <class T, int HD, int MODE, int PARTS>
void launch(cudaStream_t s, const AttnArgs& a, const AttnSplitSpace* sp) {
    using C = Cfg<HD, MODE, PARTS>;
    static std::atomic<unsigned long long> attr{0};
    once_per_device(attr, [] {
        N3D_CUDA(cudaFuncSetAttribute(attention_train_tc_kernel<T, HD, MODE, PARTS>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    });
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const int rows = MODE == GRAD_KV ? a.k_rows : a.q_rows, heads = MODE == GRAD_KV ? a.k_heads : a.q_heads;
    TcArgs t{};
    t.a = a;
    t.tiles = (rows + ROWS - 1) / ROWS;
    const long long blocks = (long long)t.tiles * heads * a.seqs;
    if (blocks > INT_MAX) throw Error(13, "attention: more than 2^31 tiles");
    if (blocks == 0) return;
    auto map = [&](const HeadsView& v, int n, int h, int box) {
        return make_heads_map(v.p, bf16, a.seqs, n, h, HD, v.seq, v.row, v.head, box);
    };
    // an operand: the tensor itself, or its pair [part][seqs][heads][rows][HD]
    auto operand = [&](const HeadsView& v, void* pair, int n, int h) {
        if (PARTS == 1) return map(v, n, h, 64);
        return make_heads_map(pair, false, 2LL * a.seqs, n, h, HD, (long long)h * n * HD, HD, (long long)n * HD, 64);
    };
    const AttnSplitSpace none{};
    const AttnSplitSpace& p = sp ? *sp : none;
    TcMaps m{};
    // a tensor without rows is never loaded: any valid map stands in for its own
    const CUtensorMap stand_in = MODE == GRAD_KV ? operand(a.k, p.k, rows, heads) : operand(a.q, p.q, rows, heads);
    m.q = a.q_rows ? operand(a.q, p.q, a.q_rows, a.q_heads) : stand_in;
    m.k = a.k_rows ? operand(a.k, p.k, a.k_rows, a.k_heads) : stand_in;
    m.v = a.k_rows ? operand(a.v, p.v, a.k_rows, a.k_heads) : stand_in;
    if (MODE != FORWARD) m.dout = a.q_rows ? operand(a.dout, p.dout, a.q_rows, a.q_heads) : stand_in;
    if (PARTS == 1 && MODE == FORWARD) m.out = map(a.o, a.q_rows, a.q_heads, 32);
    if (PARTS == 1 && MODE == GRAD_Q) m.dq = map(a.dq, a.q_rows, a.q_heads, 32);
    if (PARTS == 1 && MODE == GRAD_KV) {
        m.dk = map(a.dk, a.k_rows, a.k_heads, 32);
        m.dv = map(a.dv, a.k_rows, a.k_heads, 32);
    }
    const bool before = a.left >= kNoLimit, after = a.right >= kNoLimit;
    t.run = before != after ? (int)std::min<long long>((long long)heads * a.seqs, 32) : 1;
    t.ascending = before;
    t.k2 = fabsf(a.scale) * LOG2E;
    t.factor = a.scale;
    t.negate = a.scale < 0.0f;
    t.q_tiles = (a.q_rows + ROWS - 1) / ROWS;
    t.k_tiles = (a.k_rows + COLS - 1) / COLS;
    if (PARTS == 1) {
        t.stats = a.row_dot;
        t.norms = a.row_dot + (size_t)a.seqs * a.q_heads * t.q_tiles * 256;
    } else {
        t.stats = p.stats;
        t.key_stats = p.key_stats;
    }
    launch_pdl(attention_train_tc_kernel<T, HD, MODE, PARTS>, dim3((unsigned)blocks), dim3(C::THREADS), C::SMEM, s, m, t);
}

template <class T, int HD, int PARTS>
void launch_modes(cudaStream_t s, const AttnArgs& a, bool backward, const AttnSplitSpace* sp) {
    if (!backward) return launch<T, HD, FORWARD, PARTS>(s, a, sp);
    launch<T, HD, GRAD_Q, PARTS>(s, a, sp);
    launch<T, HD, GRAD_KV, PARTS>(s, a, sp);
}
template <class T, int PARTS>
void launch_dim(cudaStream_t s, const AttnArgs& a, bool backward, const AttnSplitSpace* sp) {
    a.head_dim == 64 ? launch_modes<T, 64, PARTS>(s, a, backward, sp) : launch_modes<T, 128, PARTS>(s, a, backward, sp);
}

// Whole 16-byte words, and strides that a tensor map can hold (above 0, below 2^40 bytes).
bool tma_view(const HeadsView& v, long long seqs, long long rows, long long heads) {
    if (rows == 0) return true;
    auto fits = [](long long st, long long n) { return n <= 1 || (st > 0 && st % 8 == 0 && st < (1LL << 39)); };
    return reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && fits(v.seq, seqs) && fits(v.row, rows) && fits(v.head, heads);
}

}  // namespace

bool attention_tc_fits(const AttnArgs& a, int dtype, bool backward) {
    if (dtype == N3D_F32) return attention_split_pays(a.q_rows, a.k_rows, backward);
    auto q_side = [&](const HeadsView& v) { return tma_view(v, a.seqs, a.q_rows, a.q_heads); };
    auto k_side = [&](const HeadsView& v) { return tma_view(v, a.seqs, a.k_rows, a.k_heads); };
    const bool f = q_side(a.q) && q_side(a.o) && k_side(a.k) && k_side(a.v);
    return f && (!backward || (q_side(a.dout) && q_side(a.dq) && k_side(a.dk) && k_side(a.dv)));
}

// The split's launch and its blocks of one per SM cost more than they save where all of a head is
// one tile of the fp32 units: forward, 32 sequences x 8 heads of 64 x 64 rows take 24 us against 18 there, 128 of
// 32 rows 65 against 52; of 65 rows 29 against 52, 8 of 128 rows 18 against 20, 8 of 256 rows 23 against 49.
// The gradient pays everywhere (1 x 16 rows 25 us against 30, 128 x 32 rows 133 against 175, 8 x 256 rows 43
// against 155).
bool attention_split_pays(size_t q_rows, size_t k_rows, bool backward) {
    return q_rows > 0 && k_rows > 0 && (backward || q_rows > 64 || k_rows > 64);
}

void launch_attention_train_tc(cudaStream_t s, const AttnArgs& a, int dtype, bool backward) {
    if (dtype == N3D_F32) {
        AttnSplitSpace sp;
        attn_split_space(a.row_dot, a.seqs, a.q_heads, a.k_heads, a.q_rows, a.k_rows, a.head_dim, backward, &sp);
        launch_attention_split(s, a, sp, backward);
        launch_dim<__half, 2>(s, a, backward, &sp);
    } else if (dtype == N3D_BF16) {
        launch_dim<__nv_bfloat16, 1>(s, a, backward, nullptr);
    } else {
        launch_dim<__half, 1>(s, a, backward, nullptr);
    }
}

}  // namespace n3d
