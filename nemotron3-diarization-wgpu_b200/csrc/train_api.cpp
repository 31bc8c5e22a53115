// extern "C" entry points of the training operators (include/n3d.h): argument checks,
// the device guard, the asynchronous timeout record, and the rotary plan.

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <mutex>

#include "api_guard.h"
#include "train.h"

using n3d::arg_check;
using n3d::guarded;

namespace {

// The caller's current device is put back when a call returns.
struct DeviceGuard {
    int before = -1, want;
    explicit DeviceGuard(int device) : want(device) {
        static const int count = [] {
            int n = 0;
            if (cudaGetDeviceCount(&n) != cudaSuccess) n = 0;
            cudaGetLastError();
            return n;
        }();
        if (count == 0) throw n3d::Error(N3D_ERR_NO_DEVICE, "no CUDA device");
        arg_check(device >= 0 && device < std::min(count, n3d::kMaxDevices), "device index out of range");
        N3D_CUDA(cudaGetDevice(&before));
        if (before != want) N3D_CUDA(cudaSetDevice(want));
    }
    ~DeviceGuard() {
        if (before >= 0 && before != want) cudaSetDevice(before);
    }
};

// The timeout record of each device: a word of mapped host memory that the kernels'
// bounded waits write, read here without waiting for the GPU.
int* train_error(int device) {
    static std::mutex mu;
    static int* words[n3d::kMaxDevices] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (!words[device]) {
        void* p = nullptr;
        N3D_CUDA(cudaHostAlloc(&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
        *static_cast<int*>(p) = 0;
        words[device] = static_cast<int*>(p);
    }
    return words[device];
}
void check_record(int* word) {
    if (__atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL) != 0)
        throw n3d::Error(N3D_ERR_TIMEOUT, "a bounded device wait of an earlier training operator gave up");
}

void check_dtype(int dtype) {
    arg_check(dtype == N3D_F32 || dtype == N3D_BF16 || dtype == N3D_F16, "unknown n3d_dtype");
}

// Largest element offset that is allowed, so that byte offsets stay inside 63 bits.
constexpr long long kMaxOffset = 1LL << 60;

// Non-negative strides whose largest offset is representable.  Outputs (`distinct`) must
// not overlap: taken by stride, each dimension steps over the whole of the ones below it.
void check_heads(const n3d_heads& t, size_t seqs, size_t rows, size_t dim, int dtype, bool distinct) {
    arg_check(t.d_data || seqs == 0 || rows == 0, "null tensor");
    arg_check(reinterpret_cast<uintptr_t>(t.d_data) % n3d::dtype_size(dtype) == 0, "tensor not aligned to its type");
    arg_check(t.heads >= 1 && t.heads <= 65535, "heads outside 1..65535");
    long long st[3] = {t.seq_stride, t.row_stride, t.head_stride};
    long long n[3] = {(long long)seqs, (long long)rows, (long long)t.heads};
    long long last = (long long)dim - 1;
    for (int i = 0; i < 3; i++) {
        arg_check(st[i] >= 0, "negative stride");
        if (n[i] > 1) {
            arg_check(st[i] <= (kMaxOffset - last) / (n[i] - 1), "strides beyond 2^60 elements");
            last += st[i] * (n[i] - 1);
        }
    }
    if (!distinct) return;
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return st[a] < st[b]; });
    long long span = (long long)dim;  // elements covered so far
    for (int i : order)
        if (n[i] > 1) {
            arg_check(st[i] >= span, "an output's elements overlap");
            span = st[i] * (n[i] - 1) + span;
        }
}

// One dimension of a row view: non-negative strides, representable offsets; the rows of
// an output do not overlap.
void check_rows(const n3d_rows& t, size_t rows, size_t cols, int dtype, bool distinct) {
    arg_check(t.d_data || rows == 0, "null matrix");
    arg_check(reinterpret_cast<uintptr_t>(t.d_data) % n3d::dtype_size(dtype) == 0, "matrix not aligned to its type");
    arg_check(t.row_stride >= 0, "negative row stride");
    if (rows > 1) {
        arg_check(t.row_stride <= kMaxOffset / (long long)rows, "row stride beyond 2^60 elements");
        arg_check(!distinct || t.row_stride >= (long long)cols, "an output's rows overlap");
    }
}
bool wide_rows(const n3d_rows* t, int dtype) {
    return !t || (reinterpret_cast<uintptr_t>(t->d_data) % (4 * n3d::dtype_size(dtype)) == 0 && t->row_stride % 4 == 0);
}
bool wide_weights(std::initializer_list<const float*> ws) {
    for (const float* w : ws)
        if (reinterpret_cast<uintptr_t>(w) % 16) return false;
    return true;
}
// `out` may be `in` itself (in place).
void check_in_place(const n3d_rows& out, const n3d_rows& in, size_t rows, const char* what) {
    if (out.d_data == in.d_data) arg_check(rows <= 1 || out.row_stride == in.row_stride, what);
}

void check_residual(const n3d_residual_config* cfg) {
    arg_check(cfg != nullptr, "residual norm: null configuration");
    arg_check(cfg->cols >= 1 && cfg->cols <= 8192, "residual norm: cols outside 1..8192");
    arg_check(cfg->rows <= (size_t)INT_MAX, "residual norm: rows beyond 2^31");
    check_dtype(cfg->residual_dtype);
    check_dtype(cfg->block_dtype);
    arg_check(cfg->residual_dtype == N3D_F32 || cfg->residual_dtype == cfg->block_dtype,
              "residual norm: the residual stream has the block's type or fp32");
    for (int n : {cfg->post_norm, cfg->pre_norm})
        arg_check(n == N3D_NORM_NONE || n == N3D_NORM_LAYER || n == N3D_NORM_RMS, "residual norm: unknown norm");
    arg_check(cfg->post_norm == N3D_NORM_NONE || cfg->post_eps > 0.0f, "residual norm: post_eps must be above 0");
    arg_check(cfg->pre_norm == N3D_NORM_NONE || cfg->pre_eps > 0.0f, "residual norm: pre_eps must be above 0");
}
n3d::ResidualArgs residual_args(const n3d_residual_config& cfg) {
    n3d::ResidualArgs a{};
    a.rows = (long long)cfg.rows;
    a.cols = (int)cfg.cols;
    a.post = cfg.post_norm;
    a.pre = cfg.pre_norm;
    a.post_eps = cfg.post_eps;
    a.pre_eps = cfg.pre_eps;
    a.scale = cfg.scale;
    a.rows_per_gate = (long long)std::min(cfg.rows_per_gate, std::max<size_t>(cfg.rows, 1));
    return a;
}
// The weights that the configuration uses; the others are not read, whatever the caller passed.
void set_weights(n3d::ResidualArgs& a, const float* post_w, const float* post_b, const float* gate, const float* pre_w,
                 const float* pre_b) {
    if (a.post != N3D_NORM_NONE) a.post_w = post_w, a.post_b = post_b;
    if (a.pre != N3D_NORM_NONE) a.pre_w = pre_w, a.pre_b = pre_b;
    if (a.rows_per_gate) a.gate = gate;
}
struct ResidualWorkspace {
    size_t sums, gate_parts;  // floats
};
ResidualWorkspace residual_workspace(size_t rows, size_t cols, bool gate) {
    ResidualWorkspace w{0, 0};
    for (bool wide : {false, true}) {
        const n3d::ResidualSplit sp = n3d::residual_split((long long)rows, (int)cols, wide);
        w.sums = std::max(w.sums, (size_t)sp.blocks * 4 * cols);
        w.gate_parts = std::max(w.gate_parts, gate ? (size_t)sp.slots * 2 * cols : 0);
    }
    w.sums = (w.sums + 3) / 4 * 4;
    return w;
}

n3d::HeadsView view(const n3d_heads& t) { return {t.d_data, t.seq_stride, t.row_stride, t.head_stride}; }

void check_attn(const n3d_attn_config* cfg) {
    arg_check(cfg != nullptr, "attention: null configuration");
    arg_check(cfg->head_dim == 64 || cfg->head_dim == 128, "attention: head_dim must be 64 or 128");
    check_dtype(cfg->dtype);
    arg_check(cfg->seqs <= (size_t)INT_MAX && cfg->q_rows <= (size_t)1 << 30 && cfg->k_rows <= (size_t)1 << 30,
              "attention: seqs beyond 2^31 or rows beyond 2^30");
    arg_check(std::isfinite(cfg->scale), "attention: scale is not finite");
    arg_check(cfg->left <= n3d::kMaxReach && cfg->right <= n3d::kMaxReach && cfg->q_offset <= n3d::kMaxReach &&
                  cfg->q_offset >= -n3d::kMaxReach,
              "attention: left, right or q_offset beyond 2^30");
}
// The tensors every attention call has; fills their views.
n3d::AttnArgs attn_args(const n3d_attn_config& cfg, const n3d_heads* q, const n3d_heads* k, const n3d_heads* v,
                        const n3d_heads* out, bool out_written, const int32_t* q_len, const int32_t* k_len) {
    arg_check(q && k && v && out, "attention: null argument");
    check_heads(*q, cfg.seqs, cfg.q_rows, cfg.head_dim, cfg.dtype, false);
    check_heads(*k, cfg.seqs, cfg.k_rows, cfg.head_dim, cfg.dtype, false);
    check_heads(*v, cfg.seqs, cfg.k_rows, cfg.head_dim, cfg.dtype, false);
    check_heads(*out, cfg.seqs, cfg.q_rows, cfg.head_dim, cfg.dtype, out_written);
    arg_check(k->heads == v->heads && q->heads == out->heads, "attention: q and out, k and v must have the same heads");
    arg_check(q->heads % k->heads == 0, "attention: the query heads must be a multiple of the key heads");
    n3d::AttnArgs a{};
    a.q = view(*q), a.k = view(*k), a.v = view(*v), a.o = view(*out);
    a.seqs = (int)cfg.seqs, a.q_rows = (int)cfg.q_rows, a.k_rows = (int)cfg.k_rows;
    a.q_heads = (int)q->heads, a.k_heads = (int)k->heads, a.head_dim = (int)cfg.head_dim;
    a.scale = cfg.scale != 0.0f ? cfg.scale : (float)(1.0 / std::sqrt((double)cfg.head_dim));
    a.left = cfg.left < 0 ? n3d::kNoLimit : (int)cfg.left;
    a.right = cfg.right < 0 ? n3d::kNoLimit : (int)cfg.right;
    a.offset = (int)cfg.q_offset;
    a.q_len = q_len, a.k_len = k_len;
    return a;
}
void check_workspace(size_t need, const void* p, size_t bytes) {
    arg_check(need == 0 || (p && bytes >= need && reinterpret_cast<uintptr_t>(p) % 16 == 0),
              "attention: a 16-byte aligned workspace of n3d_attention_workspace bytes is wanted");
}

// An output that stands where tensors do that other blocks, or later launches, still read or write.
void check_apart(const n3d_heads* out, std::initializer_list<const n3d_heads*> others, const char* what) {
    for (const n3d_heads* t : others) arg_check(!out->d_data || out->d_data != t->d_data, what);
}

void check_sizes(size_t seqs, size_t rows) {
    arg_check(seqs <= (size_t)INT_MAX && rows <= (size_t)INT_MAX, "seqs or rows beyond 2^31");
}

}  // namespace

extern "C" {

n3d_status n3d_train_status(int device) {
    return guarded([&] {
        DeviceGuard g(device);
        check_record(train_error(device));
    });
}

n3d_status n3d_rope_plan_make(const n3d_rope_config* cfg, n3d_rope_plan* plan) {
    return guarded([&] {
        arg_check(cfg && plan, "n3d_rope_plan_make: null argument");
        const size_t n = cfg->rotary_dim;
        arg_check(cfg->head_dim >= 2 && cfg->head_dim <= 256, "n3d_rope_plan_make: head_dim outside 2..256");
        arg_check(n >= 2 && n % 2 == 0 && n <= cfg->head_dim, "n3d_rope_plan_make: rotary_dim must be even, 2..head_dim");
        arg_check(cfg->layout == N3D_ROPE_HALF || cfg->layout == N3D_ROPE_INTERLEAVED, "n3d_rope_plan_make: bad layout");
        arg_check(cfg->scaling >= N3D_ROPE_PLAIN && cfg->scaling <= N3D_ROPE_YARN, "n3d_rope_plan_make: bad scaling");
        arg_check(std::isfinite(cfg->theta) && cfg->theta > 1.0, "n3d_rope_plan_make: theta must be above 1");
        const double factor = cfg->scaling == N3D_ROPE_PLAIN ? 1.0 : cfg->factor;
        arg_check(std::isfinite(factor) && factor >= 1.0, "n3d_rope_plan_make: factor must be at least 1");
        arg_check(std::isfinite(cfg->attention_factor), "n3d_rope_plan_make: attention_factor is not finite");
        double theta = cfg->theta, lo = 0.0, hi = 0.0, m = 1.0;
        if (cfg->scaling == N3D_ROPE_NTK && n > 2) theta *= std::pow(factor, (double)n / (double)(n - 2));
        if (cfg->scaling == N3D_ROPE_YARN) {
            arg_check(std::isfinite(cfg->original_length) && cfg->original_length > 0.0 && std::isfinite(cfg->beta_fast) &&
                          std::isfinite(cfg->beta_slow) && cfg->beta_slow > 0.0 && cfg->beta_fast >= cfg->beta_slow,
                      "n3d_rope_plan_make: YARN needs original_length > 0 and beta_fast >= beta_slow > 0");
            // the (fractional) pair that makes `turns` turns over the original length
            auto at = [&](double turns) {
                return (double)n * std::log(cfg->original_length / (turns * 2.0 * M_PI)) / (2.0 * std::log(theta));
            };
            lo = std::max(std::floor(at(cfg->beta_fast)), 0.0);
            hi = std::min(std::ceil(at(cfg->beta_slow)), (double)n - 1.0);
            m = 0.1 * std::log(factor) + 1.0;
        }
        n3d_rope_plan p{};
        p.head_dim = (uint32_t)cfg->head_dim;
        p.rotary_dim = (uint32_t)n;
        p.layout = cfg->layout;
        p.attention_factor = (float)(cfg->attention_factor != 0.0 ? cfg->attention_factor : m);
        for (size_t i = 0; i < n / 2; i++) {
            double f = std::pow(theta, -2.0 * (double)i / (double)n);
            if (cfg->scaling == N3D_ROPE_LINEAR) f /= factor;
            if (cfg->scaling == N3D_ROPE_YARN) {
                const double r = std::min(1.0, std::max(0.0, ((double)i - lo) / std::max(hi - lo, 1e-3)));
                f = f * (1.0 - r) + f / factor * r;
            }
            // f <= 1 radian per position, so less than a turn: the product stays below 2^64
            p.turns[i] = (uint64_t)std::llround(std::ldexp(f / (2.0 * M_PI), 62)) << 2;
        }
        *plan = p;
    });
}

n3d_status n3d_rope(int device, const n3d_rope_plan* plan, int dtype, size_t seqs, size_t rows, size_t count,
                    const n3d_heads* x, const n3d_heads* y, const int32_t* d_positions, long long first_position,
                    int transpose, void* stream) {
    return guarded([&] {
        arg_check(plan && x && y, "n3d_rope: null argument");
        arg_check(count == 1 || count == 2, "n3d_rope: count must be 1 or 2");
        arg_check(plan->head_dim >= 2 && plan->head_dim <= 256 && plan->rotary_dim >= 2 && plan->rotary_dim % 2 == 0 &&
                      plan->rotary_dim <= plan->head_dim,
                  "n3d_rope: the plan was not made by n3d_rope_plan_make");
        check_dtype(dtype);
        check_sizes(seqs, rows);
        arg_check(rows == 0 || seqs <= (size_t)INT_MAX * 32 / rows, "n3d_rope: more than 2^36 tokens");
        n3d::RopeArgs a{};
        size_t heads = 0;
        for (size_t i = 0; i < count; i++) {
            arg_check(x[i].heads == y[i].heads, "n3d_rope: x and y must have the same heads");
            check_heads(x[i], seqs, rows, plan->head_dim, dtype, false);
            check_heads(y[i], seqs, rows, plan->head_dim, dtype, true);
            a.x[i] = view(x[i]);
            a.y[i] = view(y[i]);
            a.in_place[i] = x[i].d_data == y[i].d_data;
            if (a.in_place[i])
                arg_check((seqs <= 1 || x[i].seq_stride == y[i].seq_stride) &&
                              (rows <= 1 || x[i].row_stride == y[i].row_stride) &&
                              (x[i].heads <= 1 || x[i].head_stride == y[i].head_stride),
                          "n3d_rope: in place, x and y must have the same strides");
            heads += x[i].heads;
        }
        if (count == 2) {
            const char* apart = "n3d_rope: an output stands where the other tensor or the other output does";
            check_apart(&y[0], {&x[1], &y[1]}, apart);
            check_apart(&y[1], {&x[0]}, apart);
        }
        if (seqs == 0 || rows == 0) return;
        if (count == 1) a.x[1] = a.x[0], a.y[1] = a.y[0];
        a.heads0 = (int)x[0].heads;
        a.heads = (int)heads;
        a.rows = (int)rows;
        a.tokens = (long long)seqs * (long long)rows;
        a.positions = d_positions;
        a.first = first_position;
        a.head_dim = (int)plan->head_dim;
        a.rotary_dim = (int)plan->rotary_dim;
        a.factor = plan->attention_factor;
        a.transpose = transpose != 0;
        DeviceGuard g(device);
        check_record(train_error(device));
        n3d::launch_rope((cudaStream_t)stream, a, *plan, dtype);
    });
}

n3d_status n3d_residual_norm(int device, const n3d_residual_config* cfg, const n3d_rows* x, const n3d_rows* block,
                             const float* d_post_w, const float* d_post_b, const float* d_gate, const float* d_pre_w,
                             const float* d_pre_b, const n3d_rows* r, const n3d_rows* y, void* stream) {
    return guarded([&] {
        check_residual(cfg);
        const bool pre = cfg->pre_norm != N3D_NORM_NONE;
        arg_check(x && block && r && (y || !pre), "n3d_residual_norm: null argument");
        arg_check(cfg->rows_per_gate == 0 || cfg->rows == 0 || d_gate, "n3d_residual_norm: null gate");
        check_rows(*x, cfg->rows, cfg->cols, cfg->residual_dtype, false);
        check_rows(*block, cfg->rows, cfg->cols, cfg->block_dtype, false);
        check_rows(*r, cfg->rows, cfg->cols, cfg->residual_dtype, true);
        if (pre) check_rows(*y, cfg->rows, cfg->cols, cfg->block_dtype, true);
        check_in_place(*r, *x, cfg->rows, "n3d_residual_norm: in place, r and x must have the same stride");
        if (pre) check_in_place(*y, *block, cfg->rows, "n3d_residual_norm: in place, y and block must have the same stride");
        n3d::ResidualArgs a = residual_args(*cfg);
        set_weights(a, d_post_w, d_post_b, d_gate, d_pre_w, d_pre_b);
        a.x = x->d_data, a.ld_x = x->row_stride;
        a.block = block->d_data, a.ld_block = block->row_stride;
        a.r_out = r->d_data, a.ld_r_out = r->row_stride;
        if (pre) a.y = y->d_data, a.ld_y = y->row_stride;
        a.wide = cfg->cols % 4 == 0 && wide_rows(x, cfg->residual_dtype) && wide_rows(r, cfg->residual_dtype) &&
                 wide_rows(block, cfg->block_dtype) && wide_rows(pre ? y : nullptr, cfg->block_dtype) &&
                 wide_weights({a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b});
        if (cfg->rows == 0) return;
        DeviceGuard g(device);
        check_record(train_error(device));
        n3d::launch_residual_norm((cudaStream_t)stream, a, cfg->residual_dtype, cfg->block_dtype);
    });
}

size_t n3d_residual_norm_workspace(size_t rows, size_t cols, size_t rows_per_gate) {
    if (rows > (size_t)INT_MAX || cols < 1 || cols > 8192) return 0;
    const ResidualWorkspace w = residual_workspace(rows, cols, rows_per_gate != 0);
    return (w.sums + w.gate_parts) * sizeof(float);
}

n3d_status n3d_residual_norm_grad(int device, const n3d_residual_config* cfg, const n3d_rows* block, const n3d_rows* r,
                                  const float* d_post_w, const float* d_post_b, const float* d_gate,
                                  const float* d_pre_w, const n3d_rows* dy, const n3d_rows* dr, const n3d_rows* dx,
                                  const n3d_rows* dblock, float* d_dgate, float* d_dpost_w, float* d_dpost_b,
                                  float* d_dpre_w, float* d_dpre_b, void* d_workspace, size_t workspace_bytes,
                                  void* stream) {
    return guarded([&] {
        check_residual(cfg);
        const bool pre = cfg->pre_norm != N3D_NORM_NONE, post = cfg->post_norm != N3D_NORM_NONE;
        arg_check(block && dx && dblock && (!pre || (r && dy)) && (pre || dr), "n3d_residual_norm_grad: null argument");
        arg_check(cfg->rows_per_gate == 0 || cfg->rows == 0 || d_gate, "n3d_residual_norm_grad: null gate");
        arg_check(cfg->rows_per_gate != 0 || !d_dgate, "n3d_residual_norm_grad: the gradient of a gate that is not used");
        arg_check(post || (!d_dpost_w && !d_dpost_b), "n3d_residual_norm_grad: gradients of a norm that is not used");
        arg_check(pre || (!d_dpre_w && !d_dpre_b), "n3d_residual_norm_grad: gradients of a norm that is not used");
        const size_t rows = cfg->rows, cols = cfg->cols;
        const int rt = cfg->residual_dtype, bt = cfg->block_dtype;
        check_rows(*block, rows, cols, bt, false);
        if (pre) check_rows(*r, rows, cols, rt, false);
        if (pre) check_rows(*dy, rows, cols, bt, false);
        if (dr) check_rows(*dr, rows, cols, rt, false);
        check_rows(*dx, rows, cols, rt, true);
        check_rows(*dblock, rows, cols, bt, true);
        const char* strides = "n3d_residual_norm_grad: in place, the strides must be the same";
        if (dr) check_in_place(*dx, *dr, rows, strides);
        if (pre) check_in_place(*dblock, *dy, rows, strides);
        check_in_place(*dblock, *block, rows, strides);
        const ResidualWorkspace w = residual_workspace(rows, cols, cfg->rows_per_gate != 0);
        arg_check(workspace_bytes >= (w.sums + w.gate_parts) * sizeof(float) && d_workspace &&
                      reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0,
                  "n3d_residual_norm_grad: a 16-byte aligned workspace of n3d_residual_norm_workspace bytes is wanted");
        DeviceGuard g(device);
        check_record(train_error(device));
        if (rows == 0) {  // sums over nothing
            for (float* p : {d_dpost_w, d_dpost_b, d_dpre_w, d_dpre_b})
                if (p) N3D_CUDA(cudaMemsetAsync(p, 0, cols * sizeof(float), (cudaStream_t)stream));
            return;
        }
        n3d::ResidualArgs a = residual_args(*cfg);
        set_weights(a, d_post_w, d_post_b, d_gate, d_pre_w, nullptr);
        a.block = block->d_data, a.ld_block = block->row_stride;
        if (pre) a.r = r->d_data, a.ld_r = r->row_stride, a.dy = dy->d_data, a.ld_dy = dy->row_stride;
        if (dr) a.dr = dr->d_data, a.ld_dr = dr->row_stride;
        a.dx = dx->d_data, a.ld_dx = dx->row_stride;
        a.dblock = dblock->d_data, a.ld_dblock = dblock->row_stride;
        a.dgate = d_dgate, a.dpost_w = d_dpost_w, a.dpost_b = d_dpost_b, a.dpre_w = d_dpre_w, a.dpre_b = d_dpre_b;
        a.sums = static_cast<float*>(d_workspace);
        a.gate_parts = a.sums + w.sums;
        a.wide = cols % 4 == 0 && wide_rows(block, bt) && wide_rows(dx, rt) && wide_rows(dblock, bt) &&
                 wide_rows(pre ? r : nullptr, rt) && wide_rows(pre ? dy : nullptr, bt) && wide_rows(dr, rt) &&
                 wide_weights({a.post_w, a.post_b, a.gate, a.pre_w, d_dgate});
        a.slots = n3d::residual_split(a.rows, a.cols, a.wide).slots;
        n3d::launch_residual_norm_grad((cudaStream_t)stream, a, rt, bt);
    });
}

size_t n3d_attention_workspace(const n3d_attn_config* cfg, size_t q_heads, size_t k_heads, int backward) {
    if (!cfg || q_heads > 65535 || k_heads > 65535 || cfg->seqs > (size_t)INT_MAX || cfg->q_rows > (size_t)1 << 30 ||
        cfg->k_rows > (size_t)1 << 30 || (cfg->head_dim != 64 && cfg->head_dim != 128))
        return 0;
    const size_t rows = backward ? n3d::attn_workspace_floats(cfg->seqs, q_heads, cfg->q_rows) * sizeof(float) : 0;
    if (cfg->dtype != N3D_F32 || !n3d::attention_split_pays(cfg->q_rows, cfg->k_rows, backward != 0)) return rows;
    return std::max(rows, n3d::attn_split_space(nullptr, cfg->seqs, q_heads, k_heads, cfg->q_rows, cfg->k_rows,
                                                cfg->head_dim, backward != 0, nullptr));
}

n3d_status n3d_attention_forward(int device, const n3d_attn_config* cfg, const n3d_heads* q, const n3d_heads* k,
                                 const n3d_heads* v, const int32_t* d_q_len, const int32_t* d_k_len,
                                 const n3d_heads* out, float* d_lse, void* d_workspace, size_t workspace_bytes,
                                 void* stream) {
    return guarded([&] {
        check_attn(cfg);
        n3d::AttnArgs a = attn_args(*cfg, q, k, v, out, true, d_q_len, d_k_len);
        check_apart(out, {k, v}, "n3d_attention_forward: out stands where keys or values do");
        check_workspace(n3d_attention_workspace(cfg, q->heads, k->heads, 0), d_workspace, workspace_bytes);
        a.lse = d_lse;
        a.row_dot = static_cast<float*>(d_workspace);
        if (cfg->seqs == 0 || cfg->q_rows == 0) return;
        DeviceGuard g(device);
        a.err = train_error(device);
        check_record(a.err);
        n3d::launch_attention_forward((cudaStream_t)stream, a, cfg->dtype);
    });
}

n3d_status n3d_attention_backward(int device, const n3d_attn_config* cfg, const n3d_heads* q, const n3d_heads* k,
                                  const n3d_heads* v, const n3d_heads* out, const float* d_lse, const n3d_heads* dout,
                                  const int32_t* d_q_len, const int32_t* d_k_len, const n3d_heads* dq,
                                  const n3d_heads* dk, const n3d_heads* dv, void* d_workspace, size_t workspace_bytes,
                                  void* stream) {
    return guarded([&] {
        check_attn(cfg);
        n3d::AttnArgs a = attn_args(*cfg, q, k, v, out, false, d_q_len, d_k_len);
        arg_check(dout && dq && dk && dv, "n3d_attention_backward: null argument");
        arg_check(d_lse || cfg->seqs == 0 || cfg->q_rows == 0, "n3d_attention_backward: null lse");
        check_heads(*dout, cfg->seqs, cfg->q_rows, cfg->head_dim, cfg->dtype, false);
        check_heads(*dq, cfg->seqs, cfg->q_rows, cfg->head_dim, cfg->dtype, true);
        check_heads(*dk, cfg->seqs, cfg->k_rows, cfg->head_dim, cfg->dtype, true);
        check_heads(*dv, cfg->seqs, cfg->k_rows, cfg->head_dim, cfg->dtype, true);
        arg_check(dout->heads == q->heads && dq->heads == q->heads && dk->heads == k->heads && dv->heads == k->heads,
                  "n3d_attention_backward: a gradient has other heads than its tensor");
        const char* apart = "n3d_attention_backward: a gradient stands where an input or another gradient does";
        check_apart(dq, {q, k, v, dout, dk, dv}, apart);
        check_apart(dk, {q, v, out, dout, dv}, apart);
        check_apart(dv, {q, k, out, dout}, apart);
        check_workspace(n3d_attention_workspace(cfg, q->heads, k->heads, 1), d_workspace, workspace_bytes);
        a.dout = view(*dout), a.dq = view(*dq), a.dk = view(*dk), a.dv = view(*dv);
        a.lse = const_cast<float*>(d_lse);
        a.row_dot = static_cast<float*>(d_workspace);
        if (cfg->seqs == 0) return;
        DeviceGuard g(device);
        a.err = train_error(device);
        check_record(a.err);
        n3d::launch_attention_backward((cudaStream_t)stream, a, cfg->dtype);
    });
}

}  // extern "C"
