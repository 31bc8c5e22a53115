// extern "C" entry points of the training operators (include/n3d.h): argument checks,
// the device guard, the asynchronous timeout record, and the rotary plan.

#include <algorithm>
#include <climits>
#include <cmath>
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

n3d::HeadsView view(const n3d_heads& t) { return {t.d_data, t.seq_stride, t.row_stride, t.head_stride}; }

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

}  // extern "C"
