// rec_ops.cpp -- see rec_ops.hpp.
#include "rec_ops.hpp"

#include <algorithm>
#include <cmath>
#include <string>

#include "row_arrays.hpp"

extern "C" {
extern const unsigned char fg_rec_f32_code_object_start[], fg_rec_f32_code_object_end[];
extern const unsigned char fg_rec_bf16_code_object_start[], fg_rec_bf16_code_object_end[];
extern const unsigned char fg_rec_f16_code_object_start[], fg_rec_f16_code_object_end[];
}

namespace fg {

using namespace rows;

namespace {

KernelArtifact rec_code_object(int dtype) {
    static const unsigned char* const start[3] = {fg_rec_f32_code_object_start, fg_rec_bf16_code_object_start,
                                                  fg_rec_f16_code_object_start};
    static const unsigned char* const end[3] = {fg_rec_f32_code_object_end, fg_rec_bf16_code_object_end,
                                                fg_rec_f16_code_object_end};
    KernelArtifact a;
    a.backend = BackendId::Hip;
    a.name = std::string("ferrum-gpu-rec-kernels-") + kTypes[dtype];
    a.target = "gfx950";
    a.image = start[dtype];
    a.size = (size_t)(end[dtype] - start[dtype]);
    return a;
}

// Bytes of an array of rows from which on rows are loaded and stored past the caches, which
// several such arrays would leave anyway.  us with ordinary accesses / past the caches, inputs of three sets in
// turn: 4 x 2048 x 4096 in bfloat16 70.4 / 64.0, 1 x 8192 x 2048 41.0 / 39.5, training step 4 x 1024
// x 2048 66.2 / 62.8.  All of them rows of whole lines, which no two workgroups share.
constexpr uint64_t kStreamBytes = 16 << 20;

void check_rate(const char* op, double rate) {
    if (!(rate >= 0) || !std::isfinite((float)rate))
        invalid(std::string(op) + ": rate must be a finite number, 0 or more, got " + std::to_string(rate));
}

}  // namespace

const RecurrenceKernels::Type& RecurrenceKernels::type(int t) const {
    std::lock_guard<std::mutex> lock(mu_);
    if (types_[t]) return *types_[t];
    HipBackend::bind(dev_.handle());
    const CaptureAllows allows;
    std::unique_ptr<Type> k(new Type);
    k->mod = dev_.load_or_cache(rec_code_object(t));
    for (int wide = 0; wide < 2; ++wide)
        k->step[wide] = HipBackend::get_kernel(
            k->mod, (std::string("fg_rec_step_") + kTypes[t] + (wide ? "_v4" : "_v1")).c_str());
    types_[t] = std::move(k);
    return *types_[t];
}

HipBackend::KernelHandle RecurrenceKernels::get(int dtype, const std::string& name) const {
    return HipBackend::get_kernel(type(dtype).mod, name.c_str());
}

void RecurrenceKernels::step(const HipBackend::DeviceHandle& dev, const fg_recurrence_step_args& a,
                             hipStream_t stream) const {
    const char* op = "recurrence_step";
    check_dtype(op, a.dtype);
    check_range(op, "rows", a.rows, 0, kMaxCount);
    check_range(op, "channels", a.channels, 1, kMaxRowStride);
    check_range(op, "state_rows", a.state_rows, a.slots ? 0 : a.rows, kMaxCount);
    check_rate(op, a.rate);
    const uint32_t es = kBytes[a.dtype];
    const int64_t state = size_of(op, "state", {4, a.state_rows, a.channels});
    Arrays all(op, a.rows, 1, es);
    fg_rec_step_kargs g{};
    g.x = all.rows("x", a.x, a.channels, false);
    g.ga = all.rows("gate_a", a.gate_a, a.channels, false);
    g.gx = all.rows("gate_x", a.gate_x, a.channels, false);
    g.out = all.rows("out", a.out, a.channels, true);
    all.flat("decay", a.decay, 4 * a.channels, false, false);
    all.flat("bias_a", a.bias_a, 4 * a.channels, false, true);
    all.flat("bias_x", a.bias_x, 4 * a.channels, false, true);
    all.flat("state", a.state, state, a.state_out == a.state, false);
    if (a.state_out != a.state || !a.state_out) all.flat("state_out", a.state_out, state, true, false);
    all.flat("slots", a.slots, 4 * a.rows, false, true);
    if (a.rows == 0) return;
    g.decay = a.decay;
    g.bias_a = a.bias_a;
    g.bias_x = a.bias_x;
    g.state = a.state;
    g.state_out = a.state_out;
    g.slots = a.slots;
    g.state_rows = (uint64_t)a.state_rows;
    g.rows = (uint32_t)a.rows;
    g.channels = (uint32_t)a.channels;
    g.rate = (float)a.rate;
    bool wide = g.channels % 4 == 0;
    for (const fg_ssm_view* v : {&g.x, &g.ga, &g.gx, &g.out}) wide = wide && vector_rows(*v, 4, es);
    for (const float* p : {a.decay, a.bias_a, a.bias_x, a.state, (const float*)a.state_out}) wide = wide && vector_ptr(p, 16);
    const uint64_t waves = ceil_div(g.channels / (wide ? 4 : 1), 64) * g.rows;
    void* args[] = {&g};
    launch(dev, stream, type((int)a.dtype).step[wide], ceil_div(waves, 4), 256, args, op);
}

RecurrencePlan::RecurrencePlan(const HipBackend::DeviceHandle& dev, const RecurrenceKernels& k,
                               const fg_recurrence_shape& s)
    : dev_(dev), s_(s) {
    const char* op = "recurrence plan";
    check_dtype(op, s.dtype);
    check_sequences(op, s.sequences, s.length, s.tokens, s.packed);
    check_range(op, "channels", s.channels, 1, kMaxRowStride);
    check_rate(op, s.rate);
    check_rows(op, s, s.channels);
    size_of(op, "states", {4, s.sequences, s.channels});
    chains_ = s.packed ? std::min<int64_t>(s.sequences, 1) : s.sequences;
    rows_ = s.packed ? s.tokens : s.length;
    blocks_ = (uint32_t)ceil_div(s.channels, FG_REC_CHANNELS);
    const std::string tail = std::string(kTypes[s.dtype]) + (s.packed ? "_packed" : "");
    const bool stream = (uint64_t)s.channels * rows_ * chains_ * kBytes[s.dtype] >= kStreamBytes;
    for (int wide = 0; wide < 2; ++wide) {
        const std::string form = tail + (wide ? stream ? "_stream" : "" : "_any");
        forward_[wide] = k.get((int)s.dtype, "fg_rec_" + form);
        backward_[wide] = k.get((int)s.dtype, "fg_rec_back_" + form);
    }
    reduce_ = k.get((int)s.dtype, "fg_rec_reduce");
    ahead_ = chain(false);
}

uint32_t RecurrencePlan::wave_tokens(bool back) const {
    return FG_REC_ROWS * (back ? FG_REC_BACK_SEGMENT : FG_REC_SEGMENT(kBytes[s_.dtype]));
}

// As many as the rows of a chain take.
uint32_t RecurrencePlan::waves(bool back) const {
    return (uint32_t)std::min<uint64_t>(back ? FG_REC_BACK_WAVES : FG_REC_WAVES,
                                        std::max<uint64_t>(1, ceil_div(rows_, wave_tokens(back))));
}

uint64_t RecurrencePlan::places(bool back) const {
    const uint64_t tiles = std::max<uint64_t>(1, ceil_div(rows_, wave_tokens(back) * waves(back)));
    const uint64_t n = (uint64_t)size_of("recurrence", "launch", {blocks_, (int64_t)chains_, (int64_t)tiles});
    if (n > 0xffffffffull / (64 * waves(back))) invalid("recurrence: too large for one launch");
    return n;
}

// None where every chain is one tile.
Buffer<char, HipBackend> RecurrencePlan::chain(bool back) const {
    const uint64_t n = places(back), across = blocks_ * chains_;
    if (n <= across) return {};
    return Buffer<char, HipBackend>(dev_, FG_REC_CHAIN_BYTES(across, n / across));
}

size_t RecurrencePlan::checkpoint_bytes() const {
    const uint64_t checks = ceil_div(rows_, FG_REC_CHECK);
    return 4 * (uint64_t)s_.channels * (chains_ * checks + (s_.packed ? s_.sequences : 0));
}

void RecurrencePlan::info(fg_recurrence_plan_info* out) {
    std::lock_guard<std::mutex> lock(mu_);
    out->forward_tokens = wave_tokens(false) * waves(false);
    out->backward_tokens = wave_tokens(true) * waves(true);
    out->workspace_bytes = (int64_t)(part_.bytes() + ahead_.bytes() + back_.bytes());
}

fg_rec_kargs RecurrencePlan::base(const char* op, const fg_recurrence_inputs& in, bool back) const {
    if (s_.packed && !in.offsets) invalid(std::string(op) + ": packed sequences need offsets");
    if (!s_.packed && in.offsets) invalid(std::string(op) + ": offsets are for packed sequences");
    fg_rec_kargs g{};
    g.decay = in.decay;
    g.bias_a = in.bias_a;
    g.bias_x = in.bias_x;
    g.offsets = in.offsets;
    g.tokens = rows_;
    g.checks = ceil_div(rows_, FG_REC_CHECK);
    g.seqs = (uint32_t)s_.sequences;
    g.chains = (uint32_t)chains_;
    g.channels = (uint32_t)s_.channels;
    g.blocks = blocks_;
    g.rate = (float)s_.rate;
    const uint64_t n = places(back), across = (uint64_t)g.blocks * g.chains;
    g.tiles = across ? (uint32_t)(n / across) : 1;
    g.parts = chains_ * g.tiles;
    g.chain = (unsigned long long*)(back ? back_ : ahead_).data();
    fg_rec_set_divisors(&g);
    return g;
}

void RecurrencePlan::forward(const fg_recurrence_forward_args& a, hipStream_t stream) const {
    const char* op = "recurrence forward";
    const uint32_t es = kBytes[s_.dtype];
    fg_rec_kargs g = base(op, a.in, false);
    Arrays all(op, s_.packed ? 1 : s_.sequences, rows_, es);
    const int64_t state = 4 * s_.sequences * s_.channels;
    g.x = all.rows("x", a.in.x, s_.channels, false);
    g.ga = all.rows("gate_a", a.in.gate_a, s_.channels, false);
    g.gx = all.rows("gate_x", a.in.gate_x, s_.channels, false);
    g.out = all.rows("out", a.out, s_.channels, true);
    all.flat("decay", a.in.decay, 4 * s_.channels, false, false);
    all.flat("bias_a", a.in.bias_a, 4 * s_.channels, false, true);
    all.flat("bias_x", a.in.bias_x, 4 * s_.channels, false, true);
    all.flat("initial", a.initial, state, a.initial == a.final, true);
    if (a.final != a.initial) all.flat("final", a.final, state, true, true);
    all.flat("offsets", a.in.offsets, 4 * (s_.sequences + 1), false, true);
    all.flat("checkpoints", a.checkpoints, (int64_t)checkpoint_bytes(), true, true);
    if (!chains_) return;
    g.initial = a.initial;
    g.final = a.final;
    g.check = (float*)a.checkpoints;
    bool wide = g.channels % FG_REC_LANE_CHANNELS == 0;
    for (const fg_ssm_view* v : {&g.x, &g.ga, &g.gx, &g.out}) wide = wide && vector_rows(*v, FG_REC_LANE_CHANNELS, es);
    for (const float* p : {g.decay, g.bias_a, g.bias_x, g.initial, (const float*)g.final, (const float*)g.check})
        wide = wide && vector_ptr(p, 4 * FG_REC_LANE_CHANNELS);
    void* args[] = {&g};
    launch(dev_, stream, forward_[wide], (uint64_t)g.blocks * g.chains * g.tiles, 64 * waves(false), args, op);
}

void RecurrencePlan::backward(const fg_recurrence_backward_args& a, hipStream_t stream) {
    const char* op = "recurrence backward";
    const uint32_t es = kBytes[s_.dtype];
    fg_rec_kargs g = base(op, a.in, true);
    Arrays all(op, s_.packed ? 1 : s_.sequences, rows_, es);
    const int64_t state = 4 * s_.sequences * s_.channels;
    g.x = all.rows("x", a.in.x, s_.channels, false);
    g.ga = all.rows("gate_a", a.in.gate_a, s_.channels, false);
    g.gx = all.rows("gate_x", a.in.gate_x, s_.channels, false);
    g.out = all.rows("grad_out", a.grad_out, s_.channels, false);
    g.dx = all.rows("grad_x", a.grad_x, s_.channels, true, true);
    g.dga = all.rows("grad_gate_a", a.grad_gate_a, s_.channels, true, true);
    g.dgx = all.rows("grad_gate_x", a.grad_gate_x, s_.channels, true, true);
    all.flat("decay", a.in.decay, 4 * s_.channels, false, false);
    all.flat("bias_a", a.in.bias_a, 4 * s_.channels, false, true);
    all.flat("bias_x", a.in.bias_x, 4 * s_.channels, false, true);
    all.flat("offsets", a.in.offsets, 4 * (s_.sequences + 1), false, true);
    all.flat("checkpoints", a.checkpoints, (int64_t)checkpoint_bytes(), false, false);
    all.flat("grad_final", a.grad_final, state, false, true);
    all.flat("grad_initial", a.grad_initial, state, true, true);
    all.flat("grad_decay", a.grad_decay, 4 * s_.channels, true, true);
    all.flat("grad_bias_a", a.grad_bias_a, 4 * s_.channels, true, true);
    all.flat("grad_bias_x", a.grad_bias_x, 4 * s_.channels, true, true);
    g.check = (float*)const_cast<void*>(a.checkpoints);
    g.gfinal = a.grad_final;
    g.ginitial = a.grad_initial;
    g.gdecay = a.grad_decay;
    g.gbias_a = a.grad_bias_a;
    g.gbias_x = a.grad_bias_x;
    {
        std::lock_guard<std::mutex> lock(mu_);
        if (!part_.data() && chains_) {
            refuse_capture(op, dev_, stream);
            size_of(op, "workspace", {4, 3, s_.channels, (int64_t)g.parts});
            back_ = chain(true);
            part_ = Buffer<float, HipBackend>(dev_, 3 * (uint64_t)s_.channels * g.parts);
        }
    }
    g.chain = (unsigned long long*)back_.data();
    g.part = part_.data();
    bool wide = g.channels % FG_REC_LANE_CHANNELS == 0;
    for (const fg_ssm_view* v : {&g.x, &g.ga, &g.gx, &g.out, &g.dx, &g.dga, &g.dgx}) wide = wide && vector_rows(*v, FG_REC_LANE_CHANNELS, es);
    for (const float* p : {g.decay, g.bias_a, g.bias_x, g.gfinal, (const float*)g.ginitial, (const float*)g.check})
        wide = wide && vector_ptr(p, 4 * FG_REC_LANE_CHANNELS);
    void* args[] = {&g};
    if (chains_) launch(dev_, stream, backward_[wide], (uint64_t)g.blocks * g.chains * g.tiles, 64 * waves(true), args, op);
    if (g.gdecay || g.gbias_a || g.gbias_x) launch(dev_, stream, reduce_, ceil_div(3 * (uint64_t)g.channels, 64), 1024, args, op);
}

}  // namespace fg
