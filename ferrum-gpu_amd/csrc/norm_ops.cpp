// norm_ops.cpp -- see norm_ops.hpp.
#include "norm_ops.hpp"

#include <algorithm>
#include <cmath>
#include <string>

#include "row_arrays.hpp"

extern "C" {
extern const unsigned char fg_norm_f32_code_object_start[], fg_norm_f32_code_object_end[];
extern const unsigned char fg_norm_bf16_code_object_start[], fg_norm_bf16_code_object_end[];
extern const unsigned char fg_norm_f16_code_object_start[], fg_norm_f16_code_object_end[];
}

namespace fg {

using namespace rows;

namespace {

KernelArtifact norm_code_object(int dtype) {
    static const unsigned char* const start[3] = {fg_norm_f32_code_object_start, fg_norm_bf16_code_object_start,
                                                  fg_norm_f16_code_object_start};
    static const unsigned char* const end[3] = {fg_norm_f32_code_object_end, fg_norm_bf16_code_object_end,
                                                fg_norm_f16_code_object_end};
    KernelArtifact a;
    a.backend = BackendId::Hip;
    a.name = std::string("ferrum-gpu-norm-kernels-") + kTypes[dtype];
    a.target = "gfx950";
    a.image = start[dtype];
    a.size = (size_t)(end[dtype] - start[dtype]);
    return a;
}

// Bytes of an array of rows from which on they are stored past the caches, which several
// such arrays would leave anyway: 32 M elements of dropout in bfloat16 29.5 us with ordinary stores,
// 22.1 so; 8192 x 4096 rows to 8 bits 57 and 53.
constexpr uint64_t kStreamBytes = 16 << 20;

// Threads of a launch, whose teams take row after row and load the next one meanwhile.  8192 x 4096
// rows to 8 bits 45.7 us, with twice as many 50.1, four times 47.2; a training step 120, and
// backward, where each team leaves a part of the weight's gradient, more with more.
constexpr uint32_t kThreads = 262144;

// Kept where 32 bits are at least p 2^32, to the nearest: for p of 1, never.
template <class Args>
void set_dropout(const char* op, Args& g, double p, uint64_t seed, uint64_t offset, const int64_t* counter) {
    if (!(p >= 0 && p <= 1)) invalid(std::string(op) + ": dropout must be in [0, 1], got " + std::to_string(p));
    if (reinterpret_cast<uintptr_t>(counter) % 8) invalid(std::string(op) + ": counter: not aligned to its elements");
    const uint64_t bits = (uint64_t)std::nearbyint(p * 4294967296.0);
    g.drop_all = bits >> 32;
    g.drop = g.drop_all ? 1 : (uint32_t)bits;
    g.keep = g.drop_all ? 0.0f : (float)(1 / (1 - p));
    g.seed = seed;
    g.offset = offset;
    g.counter = counter;
}

bool same(const fg_rows& a, const fg_rows& b, int64_t rows) {
    return a.ptr && a.ptr == b.ptr && (rows < 2 || a.row_stride == b.row_stride);
}

}  // namespace

const NormKernels::Type& NormKernels::type(int t) const {
    std::lock_guard<std::mutex> lock(mu_);
    if (types_[t]) return *types_[t];
    HipBackend::bind(dev_.handle());
    const CaptureAllows allows;
    std::unique_ptr<Type> k(new Type);
    k->mod = dev_.load_or_cache(norm_code_object(t));
    k->dropout = HipBackend::get_kernel(k->mod, (std::string("fg_dropout_") + kTypes[t]).c_str());
    types_[t] = std::move(k);
    return *types_[t];
}

HipBackend::KernelHandle NormKernels::get(int dtype, const std::string& name) const {
    return HipBackend::get_kernel(type(dtype).mod, name.c_str());
}

void NormKernels::dropout(const HipBackend::DeviceHandle& dev, const fg_dropout_args& a, hipStream_t stream) const {
    const char* op = "dropout";
    check_dtype(op, a.dtype);
    check_range(op, "n", a.n, 0, kMaxBytes / kBytes[a.dtype]);
    const uint32_t es = kBytes[a.dtype];
    fg_dropout_kargs g{};
    set_dropout(op, g, a.p, a.seed, a.offset, a.counter);
    Arrays all(op, 1, 1, es);
    all.flat("x", a.x, a.n * es, a.out == a.x, false, es);
    if (a.out != a.x) all.flat("out", a.out, a.n * es, true, false, es);
    all.flat("counter", a.counter, 8, false, true, 8);
    if (!a.n) return;
    g.x = a.x;
    g.out = a.out;
    g.n = (uint64_t)a.n;
    g.stream = g.n * es >= kStreamBytes;
    const uint64_t blocks = std::min<uint64_t>(ceil_div(g.n, 256 * (16 / es)), 1u << 16);
    void* args[] = {&g};
    launch(dev, stream, type((int)a.dtype).dropout, blocks, 256, args, op);
}

NormPlan::NormPlan(const HipBackend::DeviceHandle& dev, const NormKernels& k, const fg_norm_shape& s)
    : dev_(dev), s_(s) {
    const char* op = "norm plan";
    check_dtype(op, s.dtype);
    check_range(op, "rows", s.rows, 0, kMaxCount);
    check_range(op, "width", s.width, 1, kMaxRowStride);
    if (s.group != 0 && s.group != 32 && s.group != 64 && s.group != 128)
        invalid("norm plan: group must be 0, 32, 64 or 128, got " + std::to_string(s.group));
    if (!(s.eps >= 0) || !std::isfinite((float)s.eps))
        invalid("norm plan: eps must be a finite number, 0 or more, got " + std::to_string(s.eps));
    size_of(op, "rows", {s.rows, s.width, kBytes[s.dtype]});
    const uint32_t chunk = 16 / kBytes[s.dtype];
    const uint64_t chunks = ceil_div(s.width, chunk);
    // a wave for narrow rows; else a workgroup, with as few chunks of a thread as it can have
    team_ = chunks <= 128 ? 64 : chunks <= 256 ? 256 : chunks <= 512 ? 512 : 1024;
    const uint32_t c = team_ * 2 < chunks ? 0 : team_ < chunks ? 2 : 1;
    const std::string tail = std::string(kTypes[s.dtype]) + "_c" + std::to_string(c) + "_t" + std::to_string(team_) +
                             (s.width % chunk ? "_any" : "");
    forward_ = k.get((int)s.dtype, "fg_norm_" + tail);
    backward_ = k.get((int)s.dtype, "fg_norm_back_" + tail);
    reduce_ = k.get((int)s.dtype, "fg_norm_reduce");
}

void NormPlan::info(fg_norm_plan_info* out) {
    std::lock_guard<std::mutex> lock(mu_);
    out->row_threads = team_;
    out->workspace_bytes = (int64_t)part_.bytes();
}

uint32_t NormPlan::teams() const { return FG_NORM_THREADS(team_) / team_; }

uint64_t NormPlan::workgroups(uint64_t rows) const {
    return std::min<uint64_t>(ceil_div(rows, teams()), kThreads / FG_NORM_THREADS(team_));
}

fg_norm_kargs NormPlan::base(const char* op, int64_t rows, const float* weight, double dropout, uint64_t seed,
                             uint64_t offset, const int64_t* counter) const {
    if (rows < 0 || rows > s_.rows)
        invalid(std::string(op) + ": rows must be in [0, " + std::to_string(s_.rows) + "], the plan's, got " +
                std::to_string(rows));
    fg_norm_kargs g{};
    set_dropout(op, g, dropout, seed, offset, counter);
    g.weight = weight;
    g.rows = (uint64_t)rows;
    g.width = (uint32_t)s_.width;
    g.stream = g.rows * g.width * kBytes[s_.dtype] >= kStreamBytes;
    g.groups = s_.group ? (uint32_t)ceil_div(s_.width, s_.group) : 1;
    g.group_lanes = (uint32_t)s_.group / (16 / kBytes[s_.dtype]);
    g.eps = (float)s_.eps;
    g.over_width = (float)(1.0 / s_.width);
    return g;
}

void NormPlan::forward(const fg_norm_forward_args& a, hipStream_t stream) const {
    const char* op = "norm forward";
    const uint32_t es = kBytes[s_.dtype];
    fg_norm_kargs g = base(op, a.rows, a.weight, a.dropout, a.seed, a.offset, a.counter);
    // out may be x and sum the residual: every element is read before its place is written
    const bool over_x = !a.scales && same(a.out, a.x, a.rows), over_residual = same(a.sum, a.residual, a.rows);
    Arrays all(op, 1, a.rows, es);
    g.x = all.rows("x", a.x, s_.width, over_x);
    g.residual = all.rows("residual", a.residual, s_.width, over_residual, true);
    g.out = over_x ? g.x : all.rows("out", a.out, s_.width, true, false, a.scales ? 1 : 0);
    g.sum = over_residual ? g.residual : all.rows("sum", a.sum, s_.width, true, true);
    all.flat("weight", a.weight, 4 * s_.width, false, true);
    all.flat("scales", a.scales, 4 * a.rows * g.groups, true, true);
    all.flat("counter", a.counter, 8, false, true, 8);
    if (a.rows == 0) return;
    g.scales = a.scales;
    void* args[] = {&g};
    launch(dev_, stream, forward_, workgroups(g.rows), FG_NORM_THREADS(team_), args, op);
}

void NormPlan::backward(const fg_norm_backward_args& a, hipStream_t stream) {
    const char* op = "norm backward";
    const uint32_t es = kBytes[s_.dtype];
    fg_norm_kargs g = base(op, a.rows, a.weight, a.dropout, a.seed, a.offset, a.counter);
    const bool over_sum = same(a.grad_residual, a.grad_sum, a.rows), over_out = same(a.grad_x, a.grad_out, a.rows);
    Arrays all(op, 1, a.rows, es);
    g.x = all.rows("sum", a.sum, s_.width, false);
    g.out = all.rows("grad_out", a.grad_out, s_.width, over_out);
    g.residual = all.rows("grad_sum", a.grad_sum, s_.width, over_sum, true);
    g.dx = over_out ? g.out : all.rows("grad_x", a.grad_x, s_.width, true, true);
    g.dresidual = over_sum ? g.residual : all.rows("grad_residual", a.grad_residual, s_.width, true, true);
    all.flat("weight", a.weight, 4 * s_.width, false, true);
    all.flat("grad_weight", a.grad_weight, 4 * s_.width, true, true);
    all.flat("counter", a.counter, 8, false, true, 8);
    const uint64_t blocks = workgroups(g.rows), parts = blocks * teams();
    if (a.grad_weight) {
        std::lock_guard<std::mutex> lock(mu_);
        if (!part_.data() && s_.rows) {
            refuse_capture(op, dev_, stream);
            part_ = Buffer<float, HipBackend>(
                dev_, workgroups((uint64_t)s_.rows) * teams() * (uint64_t)s_.width);
        }
        g.part = part_.data();
    }
    void* args[] = {&g};
    launch(dev_, stream, backward_, blocks, FG_NORM_THREADS(team_), args, op);
    if (a.grad_weight) {
        uint32_t n = (uint32_t)parts;
        float* to = a.grad_weight;
        void* rargs[] = {&g.part, &to, &g.width, &n};
        launch(dev_, stream, reduce_, ceil_div(g.width, 64), 1024, rargs, op);
    }
}

}  // namespace fg
