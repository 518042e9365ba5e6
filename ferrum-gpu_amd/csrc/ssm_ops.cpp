// ssm_ops.cpp -- see ssm_ops.hpp.
#include "ssm_ops.hpp"

#include <algorithm>
#include <initializer_list>
#include <string>

#include "row_arrays.hpp"

extern "C" {
extern const unsigned char fg_ssm_f32_code_object_start[], fg_ssm_f32_code_object_end[];
extern const unsigned char fg_ssm_bf16_code_object_start[], fg_ssm_bf16_code_object_end[];
extern const unsigned char fg_ssm_f16_code_object_start[], fg_ssm_f16_code_object_end[];
}

namespace fg {

using namespace rows;

namespace {

KernelArtifact ssm_code_object(int dtype) {
    static const unsigned char* const start[3] = {fg_ssm_f32_code_object_start, fg_ssm_bf16_code_object_start,
                                                  fg_ssm_f16_code_object_start};
    static const unsigned char* const end[3] = {fg_ssm_f32_code_object_end, fg_ssm_bf16_code_object_end,
                                                fg_ssm_f16_code_object_end};
    KernelArtifact a;
    a.backend = BackendId::Hip;
    a.name = std::string("ferrum-gpu-ssm-kernels-") + kTypes[dtype];
    a.target = "gfx950";
    a.image = start[dtype];
    a.size = (size_t)(end[dtype] - start[dtype]);
    return a;
}

// Channels of a thread of the convolution, widest first.
const uint32_t kVector[3] = {8, 4, 1};
// The widest of forward calls and steps: 16 bytes, and weights that fit the registers.
uint32_t conv_widest(uint32_t es, uint32_t width) { return es == 2 && width <= 4 ? 8 : 4; }

// The widest of kVector, at most `most`, that channels, rows and states allow,
// as its index.
int conv_vector(uint32_t channels, uint32_t es, std::initializer_list<const fg_ssm_view*> rows,
                std::initializer_list<const void*> states, uint32_t most) {
    for (int i = 0; i < 2; ++i) {
        const uint32_t n = kVector[i];
        bool yes = n <= most && channels % n == 0;
        for (const fg_ssm_view* v : rows) yes = yes && vector_rows(*v, n, es);
        for (const void* p : states) yes = yes && vector_ptr(p, n * es);
        if (yes) return i;
    }
    return 2;
}

}  // namespace

const SsmKernels::Type& SsmKernels::type(int t) const {
    std::lock_guard<std::mutex> lock(mu_);
    if (types_[t]) return *types_[t];
    HipBackend::bind(dev_.handle());
    const CaptureAllows allows;
    std::unique_ptr<Type> k(new Type);
    k->mod = dev_.load_or_cache(ssm_code_object(t));
    const auto find = [&](const std::string& name) { return HipBackend::get_kernel(k->mod, name.c_str()); };
    for (int w = 2; w <= FG_CONV_MAX_WIDTH; ++w)
        for (int v = 0; v < 3; ++v)
            if (kVector[v] <= conv_widest(kBytes[t], w))
                k->conv_step[w][v] = find(std::string("fg_conv_step_") + kTypes[t] + "_w" + std::to_string(w) + "_v" +
                                          std::to_string(kVector[v]));
    for (int l = 0; l < 5; ++l)
        for (int wide = 0; wide < 2; ++wide)
            k->scan_step[l][wide] = find(std::string("fg_scan_step_") + kTypes[t] + "_l" + std::to_string(1 << l) +
                                         (wide ? "" : "_any"));
    types_[t] = std::move(k);
    return *types_[t];
}

HipBackend::KernelHandle SsmKernels::get(int dtype, const std::string& name) const {
    return HipBackend::get_kernel(type(dtype).mod, name.c_str());
}

void SsmKernels::conv_step(const HipBackend::DeviceHandle& dev, const fg_conv_step_args& a,
                           hipStream_t stream) const {
    const char* op = "conv_step";
    check_dtype(op, a.dtype);
    check_range(op, "rows", a.rows, 0, kMaxCount);
    check_range(op, "channels", a.channels, 1, kMaxCount);
    check_range(op, "width", a.width, 2, FG_CONV_MAX_WIDTH);
    check_range(op, "state_rows", a.state_rows, a.slots ? 0 : a.rows, kMaxCount);
    const uint32_t es = kBytes[a.dtype];
    const int64_t state = size_of(op, "state", {a.state_rows, a.width - 1, a.channels, es});
    Arrays all(op, a.rows, 1, es);
    fg_conv_step_kargs g{};
    g.x = all.rows("x", a.x, a.channels, false);
    g.out = all.rows("out", a.out, a.channels, true);
    all.flat("weight", a.weight, 4 * a.channels * a.width, false, false);
    all.flat("bias", a.bias, 4 * a.channels, false, true);
    all.flat("state", a.state, state, a.state_out == a.state, false, es);
    if (a.state_out != a.state || !a.state_out) all.flat("state_out", a.state_out, state, true, false, es);
    all.flat("slots", a.slots, 4 * a.rows, false, true);
    if (a.rows == 0) return;
    g.weight = a.weight;
    g.bias = a.bias;
    g.state = a.state;
    g.state_out = a.state_out;
    g.slots = a.slots;
    g.state_rows = (uint64_t)a.state_rows;
    g.rows = (uint32_t)a.rows;
    g.channels = (uint32_t)a.channels;
    g.silu = a.silu != 0;
    const int v = conv_vector(g.channels, es, {&g.x, &g.out}, {a.state, a.state_out},
                              conv_widest(es, (uint32_t)a.width));
    // rows of a wave, at least 2048 waves: 256 rows x 4096 channels 6.0 us with
    // 1024 waves, 5.8 with 2048
    const uint64_t wide = ceil_div(g.channels / kVector[v], 64);
    g.each_wave = (uint32_t)std::min<uint64_t>(8, std::max<uint64_t>(1, wide * g.rows / 2048));
    const uint64_t waves = wide * ceil_div(g.rows, g.each_wave);
    void* args[] = {&g};
    launch(dev, stream, type((int)a.dtype).conv_step[a.width][v], ceil_div(waves, 4), 256, args, op);
}

void SsmKernels::scan_step(const HipBackend::DeviceHandle& dev, const fg_scan_step_args& a,
                           hipStream_t stream) const {
    const char* op = "scan_step";
    check_dtype(op, a.dtype);
    check_range(op, "rows", a.rows, 0, kMaxCount);
    check_range(op, "channels", a.channels, 1, kMaxRowStride);
    check_range(op, "states", a.states, 1, FG_SSM_MAX_STATES);
    check_range(op, "groups", a.groups, 1, a.channels);
    if (a.channels % a.groups) invalid("scan_step: groups must divide channels");
    check_range(op, "state_rows", a.state_rows, a.slots ? 0 : a.rows, kMaxCount);
    const int64_t state = size_of(op, "state", {4, a.state_rows, a.channels, a.states});
    Arrays all(op, a.rows, 1, kBytes[a.dtype]);
    fg_scan_step_kargs g{};
    g.u = all.rows("u", a.u, a.channels, false);
    g.delta = all.rows("delta", a.delta, a.channels, false);
    g.b = all.rows("B", a.b, a.groups * a.states, false);
    g.c = all.rows("C", a.c, a.groups * a.states, false);
    g.z = all.rows("z", a.z, a.channels, false, true);
    g.out = all.rows("out", a.out, a.channels, true);
    all.flat("A", a.a, 4 * a.channels * a.states, false, false);
    all.flat("D", a.d, 4 * a.channels, false, true);
    all.flat("delta_bias", a.delta_bias, 4 * a.channels, false, true);
    all.flat("state", a.state, state, a.state_out == a.state, false);
    if (a.state_out != a.state || !a.state_out) all.flat("state_out", a.state_out, state, true, false);
    all.flat("slots", a.slots, 4 * a.rows, false, true);
    if (a.rows == 0) return;
    g.a = a.a;
    g.skip = a.d;
    g.bias = a.delta_bias;
    g.state = a.state;
    g.state_out = a.state_out;
    g.slots = a.slots;
    g.state_rows = (uint64_t)a.state_rows;
    g.rows = (uint32_t)a.rows;
    g.channels = (uint32_t)a.channels;
    g.states = (uint32_t)a.states;
    g.groups = (uint32_t)a.groups;
    g.group_channels = g.channels / g.groups;
    int lanes = 0;  // log2
    while (4u << lanes < g.states) ++lanes;
    g.softplus = a.softplus != 0;
    const bool wide = g.states == 4u << lanes && vector_rows(g.b, 4, kBytes[a.dtype]) &&
                      vector_rows(g.c, 4, kBytes[a.dtype]) && vector_ptr(a.a, 16) && vector_ptr(a.state, 16) &&
                      vector_ptr(a.state_out, 16);
    // rows of a wave, at least 8192 waves, as many as are resident: 256 rows x
    // 4096 channels x 16 states 40 us with 4096, 34 with 8192, 35 with 16384
    const uint64_t per_row = ceil_div((uint64_t)g.channels << lanes, 64);
    g.each_wave = (uint32_t)std::min<uint64_t>(16, std::max<uint64_t>(1, per_row * g.rows / 8192));
    const uint64_t waves = per_row * ceil_div(g.rows, g.each_wave);
    void* args[] = {&g};
    launch(dev, stream, type((int)a.dtype).scan_step[lanes][wide], ceil_div(waves, 4), 256, args, op);
}

// ------------------------------------------------------------- convolution

namespace {

// Waves that a thread's run of tokens may leave: longer runs read fewer rows
// twice and bring fewer parts to sum, shorter ones keep more loads on their way.
// Measured, us for 1024 / 2048 / 4096 waves: forward, 9 packed sequences, 9001
// tokens x 1536 channels in float16 18.2 / 14.4 / 14.9, 8 x 2048 tokens x 4096
// channels in bfloat16 (runs of 64 and 64 / 32) - / 50.6 / 55.0.  Backward, the
// last with 4096 / 8192 waves: 104 and 8.0 for the sums / 120 and 13.6.
constexpr uint32_t kConvForwardWaves = 2048, kConvBackwardWaves = 4096;

}  // namespace

ConvPlan::ConvPlan(const HipBackend::DeviceHandle& dev, const SsmKernels& k, const fg_conv_shape& s)
    : dev_(dev), s_(s) {
    const char* op = "conv plan";
    check_dtype(op, s.dtype);
    check_sequences(op, s.sequences, s.length, s.tokens, s.packed);
    check_range(op, "channels", s.channels, 1, kMaxCount);
    check_range(op, "width", s.width, 2, FG_CONV_MAX_WIDTH);
    check_rows(op, s, s.channels);
    size_of(op, "states", {s.sequences, s.width - 1, s.channels, kBytes[s.dtype]});
    if (!s_.packed) s_.tokens = s_.sequences * s_.length;
    const std::string type = kTypes[s.dtype], w = "_w" + std::to_string(s.width);
    for (int v = 0; v < 3; ++v) {
        const std::string tail = type + w + "_v" + std::to_string(kVector[v]);
        if (kVector[v] <= conv_widest(kBytes[s.dtype], (uint32_t)s.width)) forward_[v] = k.get((int)s.dtype, "fg_conv_" + tail);
        if (kVector[v] <= 4) backward_[v] = k.get((int)s.dtype, "fg_conv_back_" + tail);
    }
    reduce_ = k.get((int)s.dtype, "fg_conv_reduce");
}

// Tokens of a thread: as many as leave `waves` waves, each of 64 threads of n
// channels, up to 64 and `least` or more.  Forward that is one group of rows (2
// x 1001 tokens x 2048 channels in bfloat16: 8.2 us, two groups 8.6) or the two
// that hold a wider window, backward two, for which half as many parts are summed.
uint32_t ConvPlan::run_for(uint32_t n, uint32_t waves, uint32_t least) const {
    const uint64_t all = ceil_div(s_.channels / n, 64) * (uint64_t)s_.tokens;
    uint32_t run = least;
    while (run < 64 && all / (2 * run) >= waves) run *= 2;
    return run;
}

// No shorter than the window: only a sequence's first run, which writes the
// final state, reads the initial one, which may be the same array.
uint32_t ConvPlan::forward_run(uint32_t n) const {
    return run_for(n, kConvForwardWaves, s_.width - 1 > FG_CONV_ROWS ? 2 * FG_CONV_ROWS : FG_CONV_ROWS);
}

// The run, and with it the workspace, is that of four channels for any call.
uint32_t ConvPlan::backward_run() const {
    return run_for(std::min<uint32_t>(4, (uint32_t)s_.channels), kConvBackwardWaves, 2 * FG_CONV_ROWS);
}

void ConvPlan::info(fg_conv_plan_info* out) {
    std::lock_guard<std::mutex> lock(mu_);
    const int v = conv_vector((uint32_t)s_.channels, 1, {}, {}, conv_widest(kBytes[s_.dtype], (uint32_t)s_.width));
    out->forward_tokens = forward_run(kVector[v]);
    out->backward_tokens = backward_run();
    out->workspace_bytes = (int64_t)part_.bytes();
}

fg_conv_kargs ConvPlan::base(const int32_t* offsets) const {
    if (s_.packed && !offsets) invalid("conv: packed sequences need offsets");
    if (!s_.packed && offsets) invalid("conv: offsets are for packed sequences");
    fg_conv_kargs g{};
    g.offsets = offsets;
    g.tokens = (uint64_t)s_.tokens;
    g.seqs = (uint32_t)s_.sequences;
    g.length = (uint32_t)s_.length;
    g.channels = (uint32_t)s_.channels;
    g.silu = s_.silu != 0;
    return g;
}

void ConvPlan::forward(const fg_conv_forward_args& a, hipStream_t stream) const {
    const char* op = "conv forward";
    const uint32_t es = kBytes[s_.dtype];
    fg_conv_kargs g = base(a.offsets);
    Arrays all(op, s_.packed ? 1 : s_.sequences, s_.packed ? s_.tokens : s_.length, es);
    g.x = all.rows("x", a.x, s_.channels, false);
    g.out = all.rows("out", a.out, s_.channels, true);
    all.flat("weight", a.weight, 4 * s_.channels * s_.width, false, false);
    all.flat("bias", a.bias, 4 * s_.channels, false, true);
    const int64_t state = s_.sequences * (s_.width - 1) * s_.channels * es;
    all.flat("initial", a.initial, state, a.initial == a.final, true, es);
    if (a.final != a.initial) all.flat("final", a.final, state, true, true, es);
    all.flat("offsets", a.offsets, 4 * (s_.sequences + 1), false, true);
    if (s_.sequences == 0) return;
    g.weight = a.weight;
    g.bias = a.bias;
    g.initial = a.initial;
    g.final = a.final;
    const int v = conv_vector(g.channels, es, {&g.x, &g.out}, {a.initial, a.final},
                              conv_widest(es, (uint32_t)s_.width));
    g.run = forward_run(kVector[v]);
    g.runs = (uint32_t)std::max<uint64_t>(1, ceil_div(g.length, g.run));
    const int64_t waves = size_of(op, "launch", {(int64_t)ceil_div(g.channels / kVector[v], 64), g.runs, g.seqs});
    void* args[] = {&g};
    launch(dev_, stream, forward_[v], ceil_div(waves, 4), 256, args, op);
}

void ConvPlan::backward(const fg_conv_backward_args& a, hipStream_t stream) {
    const char* op = "conv backward";
    const uint32_t es = kBytes[s_.dtype];
    fg_conv_kargs g = base(a.offsets);
    Arrays all(op, s_.packed ? 1 : s_.sequences, s_.packed ? s_.tokens : s_.length, es);
    g.x = all.rows("x", a.x, s_.channels, false);
    g.out = all.rows("grad_out", a.grad_out, s_.channels, false);
    g.gx = all.rows("grad_x", a.grad_x, s_.channels, true, true);
    all.flat("weight", a.weight, 4 * s_.channels * s_.width, false, false);
    all.flat("bias", a.bias, 4 * s_.channels, false, true);
    const int64_t state = s_.sequences * (s_.width - 1) * s_.channels * es;
    all.flat("initial", a.initial, state, false, true, es);
    all.flat("grad_final", a.grad_final, state, false, true, es);
    all.flat("grad_initial", a.grad_initial, state, true, true, es);
    all.flat("grad_weight", a.grad_weight, 4 * s_.channels * s_.width, true, true);
    all.flat("grad_bias", a.grad_bias, 4 * s_.channels, true, true);
    all.flat("offsets", a.offsets, 4 * (s_.sequences + 1), false, true);
    g.weight = a.weight;
    g.bias = a.bias;
    g.initial = a.initial;
    g.gfinal = a.grad_final;
    g.ginitial = a.grad_initial;
    const int v = conv_vector(g.channels, es, {&g.x, &g.out, &g.gx}, {a.initial, a.grad_final, a.grad_initial}, 4);
    g.run = backward_run();
    g.runs = (uint32_t)std::max<uint64_t>(1, ceil_div(g.length, g.run));
    const uint64_t n = (uint64_t)s_.channels * (s_.width + 1);
    {
        std::lock_guard<std::mutex> lock(mu_);
        if (!part_.data() && g.seqs) {
            refuse_capture(op, dev_, stream);
            const uint64_t places = s_.packed ? g.tokens / g.run + g.seqs : (uint64_t)g.runs * g.seqs;
            size_of(op, "workspace", {4, (int64_t)n, (int64_t)places});
            part_ = Buffer<float, HipBackend>(dev_, n * places);
        }
    }
    g.part = part_.data();
    const int64_t waves = size_of(op, "launch", {(int64_t)ceil_div(g.channels / kVector[v], 64), g.runs, g.seqs});
    void* args[] = {&g};
    launch(dev_, stream, backward_[v], ceil_div(waves, 4), 256, args, op);
    uint32_t width = (uint32_t)s_.width;
    float *gw = a.grad_weight, *gb = a.grad_bias;
    void* rargs[] = {&g, &width, &gw, &gb};
    if (gw || gb) launch(dev_, stream, reduce_, ceil_div(n, 64), 256, rargs, op);
}

// -------------------------------------------------------------------- scan

ScanPlan::ScanPlan(const HipBackend::DeviceHandle& dev, const SsmKernels& k, const fg_scan_shape& s)
    : dev_(dev), s_(s) {
    const char* op = "scan plan";
    check_dtype(op, s.dtype);
    check_sequences(op, s.sequences, s.length, s.tokens, s.packed);
    check_range(op, "channels", s.channels, 1, kMaxRowStride);
    check_range(op, "states", s.states, 1, FG_SSM_MAX_STATES);
    check_range(op, "groups", s.groups, 1, s.channels);
    if (s.channels % s.groups) invalid("scan plan: groups must divide channels");
    check_range(op, "groups * states", s.groups * s.states, 1, kMaxRowStride);
    check_rows(op, s, std::max(s.channels, s.groups * s.states));
    size_of(op, "states", {4, s.sequences, s.channels, s.states});
    if (!s_.packed) s_.tokens = s_.sequences * s_.length;
    segment_ = FG_SSM_SEGMENT;
    lane_states_ = s.states <= 4 ? 1 : s.states <= 8 ? 2 : 4;
    waves_ = s.states <= 16 ? 1 : s.states <= 32 ? 2 : 4;
    threads_ = 64 * waves_ * FG_SSM_BLOCKS(waves_);
    group_blocks_ = (uint32_t)ceil_div(s.channels / s.groups, 16 * FG_SSM_BLOCKS(waves_));
    blocks_ = group_blocks_ * (uint32_t)s.groups;
    cut(ahead_, chunks_for(512));
    cut(back_, chunks_for(s.packed ? 1536 : 1024));
    allocate(ahead_);
    const std::string type = kTypes[s.dtype];
    for (int wide = 0; wide < 2; ++wide) {
        if (wide && s.states != 4 * lane_states_ * waves_) continue;
        const std::string tail = type + "_s" + std::to_string(lane_states_) + "w" + std::to_string(waves_) +
                                 (wide ? "" : "_any");
        local_[wide] = k.get((int)s.dtype, "fg_scan_local_" + tail);
        forward_[wide] = k.get((int)s.dtype, "fg_scan_" + tail);
        back_local_[wide] = k.get((int)s.dtype, "fg_scan_back_local_" + tail);
        backward_[wide] = k.get((int)s.dtype, "fg_scan_back_" + tail);
    }
    reduce_bc_ = k.get((int)s.dtype, "fg_scan_reduce_bc_" + type);
    reduce_p_ = k.get((int)s.dtype, "fg_scan_reduce_p");
}

// Parts of the token axis that are worked through at the same time.  A SIMD of
// the GPU's 1024 takes two waves: tensors with at most `few` waves are cut
// until there are 2048 (packed ones, which count as so many of the longest's
// length, 4096: that evens unequal sequences out), into 64 parts at most, of 32
// tokens or more.  That costs a pass over the tokens for what each part adds to
// the states.  Measured, us not cut / cut so, 1024 tokens x 2048 channels x 16
// states in bfloat16 for each sequence:
//   waves              512       640       768       1024      1280      1536      1792
//   forward            83 / 71   83 / 97   84 / 111  84 / 129  -         -         -
//   backward           307 / 155 309 / 227 310 / 278 314 / 293 440 / 434 443 / 440 450 / 523
//   backward, packed   307 / 178 -         -         385 / 305 434 / 389 473 / 466 501 / 520
// Packed, 2048 / 4096: 7 sequences, 9001 tokens x 1536 channels x 8 states in
// float16, forward 136 / 97 (of an earlier kernel).  float32 backward 1152 waves 451 / 468, 300 tokens 1536 waves 141 / 149.  A part's
// least tokens, 16 / 32 / 64: forward, 300 x 1024 15.5 / 14.2 / 17.9, training step
// 128 x 1024 34 / 41 / 56, 1024 x 512 59 / 51 / 61.
uint32_t ScanPlan::chunks_for(uint32_t few) const {
    const uint64_t seqs = s_.packed && s_.length ? ceil_div(s_.tokens, s_.length) : s_.sequences;
    const uint64_t waves = std::max<uint64_t>(1, seqs * blocks_ * FG_SSM_BLOCKS(waves_) * waves_);
    if (waves > few) return 1;
    const uint64_t most = std::max<uint64_t>(1, ceil_div(s_.length, 2 * segment_));
    return (uint32_t)std::min<uint64_t>({ceil_div(s_.packed ? 4096 : 2048, waves), most, 64});
}

// Chunks of whole segments, at most `chunks` of a sequence, and their places:
// packed, one for every chunk's length of rows and one more for each sequence.
void ScanPlan::cut(Carry& c, uint32_t chunks) const {
    c.chunk_len = (uint32_t)std::max<uint64_t>(1, ceil_div(ceil_div(s_.length, chunks), segment_)) * segment_;
    c.chunks = (uint32_t)std::max<uint64_t>(1, ceil_div(s_.length, c.chunk_len));
    c.places = s_.packed ? (uint64_t)s_.tokens / c.chunk_len + s_.sequences : (uint64_t)s_.sequences * c.chunks;
}

void ScanPlan::allocate(Carry& c) const {
    if (c.chunks == 1) return;
    const int64_t sets = (int64_t)blocks_ * FG_SSM_BLOCKS(waves_);
    size_of("scan", "workspace", {4, (int64_t)c.places + s_.sequences, sets, waves_, 64, lane_states_});
    c.states = Buffer<float, HipBackend>(dev_, (c.places + s_.sequences) * sets * waves_ * 64 * lane_states_);
    c.dt = Buffer<float, HipBackend>(dev_, c.places * sets * 16);
}

void ScanPlan::info(fg_scan_plan_info* out) {
    std::lock_guard<std::mutex> lock(mu_);
    out->forward_parts = ahead_.chunks;
    out->forward_tokens = ahead_.chunk_len;
    out->backward_parts = back_.chunks;
    out->backward_tokens = back_.chunk_len;
    out->workspace_bytes = (int64_t)(ahead_.states.bytes() + ahead_.dt.bytes() + back_.states.bytes() +
                                     back_.dt.bytes() + part_bc_.bytes() + part_p_.bytes());
}

size_t ScanPlan::checkpoint_bytes() const {
    const uint64_t segs = s_.packed ? (uint64_t)s_.tokens / segment_ + s_.sequences
                                    : s_.sequences * ceil_div(s_.length, segment_);
    return segs * blocks_ * FG_SSM_BLOCKS(waves_) * waves_ * 64 * lane_states_ * sizeof(float);
}

fg_scan_kargs ScanPlan::base(const fg_scan_inputs& in, const Carry& c) const {
    fg_scan_kargs g{};
    g.a = in.a;
    g.skip = in.d;
    g.bias = in.delta_bias;
    g.initial = in.initial;
    g.offsets = in.offsets;
    g.carry = c.states.data();
    g.carry_dt = c.dt.data();
    g.tokens = (uint64_t)s_.tokens;
    g.seqs = (uint32_t)s_.sequences;
    g.length = (uint32_t)s_.length;
    g.channels = (uint32_t)s_.channels;
    g.states = (uint32_t)s_.states;
    g.groups = (uint32_t)s_.groups;
    g.group_channels = g.channels / g.groups;
    g.group_blocks = group_blocks_;
    g.chunk_len = c.chunk_len;
    g.chunks = c.chunks;
    g.places = c.places;
    g.check_segs = (uint32_t)ceil_div(s_.length, segment_);
    g.softplus = s_.softplus != 0;
    return g;
}

void ScanPlan::check_inputs(const char* op, const fg_scan_inputs& in) const {
    if (s_.packed && !in.offsets) invalid(std::string(op) + ": packed sequences need offsets");
    if (!s_.packed && in.offsets) invalid(std::string(op) + ": offsets are for packed sequences");
}

// Vector accesses where every row and every lane's part of it allow them: 4 /
// waves channels, and the lane's states of a channel that has all of them.
bool ScanPlan::wide(const fg_scan_kargs& g, std::initializer_list<const fg_ssm_view*> channels,
                    std::initializer_list<const fg_ssm_view*> states) const {
    const uint32_t es = kBytes[s_.dtype], n = 4 / waves_;
    bool yes = g.group_channels % n == 0 && g.states == 4 * lane_states_ * waves_;
    for (const fg_ssm_view* v : channels) yes = yes && vector_rows(*v, n, es);
    for (const fg_ssm_view* v : states) yes = yes && vector_rows(*v, lane_states_, es);
    return yes;
}

void ScanPlan::forward(const fg_scan_forward_args& a, hipStream_t stream) const {
    const char* op = "scan forward";
    const fg_scan_inputs& in = a.in;
    check_inputs(op, in);
    fg_scan_kargs g = base(in, ahead_);
    Arrays all(op, s_.packed ? 1 : s_.sequences, s_.packed ? s_.tokens : s_.length, kBytes[s_.dtype]);
    const int64_t state = 4 * s_.sequences * s_.channels * s_.states;
    g.u = all.rows("u", in.u, s_.channels, false);
    g.delta = all.rows("delta", in.delta, s_.channels, false);
    g.b = all.rows("B", in.b, s_.groups * s_.states, false);
    g.c = all.rows("C", in.c, s_.groups * s_.states, false);
    g.z = all.rows("z", in.z, s_.channels, false, true);
    g.out = all.rows("out", a.out, s_.channels, true);
    all.flat("A", in.a, 4 * s_.channels * s_.states, false, false);
    all.flat("D", in.d, 4 * s_.channels, false, true);
    all.flat("delta_bias", in.delta_bias, 4 * s_.channels, false, true);
    all.flat("initial", in.initial, state, in.initial == a.final, true);
    if (a.final != in.initial) all.flat("final", a.final, state, true, true);
    all.flat("offsets", in.offsets, 4 * (s_.sequences + 1), false, true);
    all.flat("checkpoints", a.checkpoints, (int64_t)checkpoint_bytes(), true, true);
    g.final = a.final;
    g.check = (float*)a.checkpoints;
    const bool vec = wide(g, {&g.u, &g.delta, &g.z, &g.out}, {&g.b, &g.c});
    void* args[] = {&g};
    const uint64_t blocks = (uint64_t)g.seqs * g.chunks * blocks_;
    if (g.chunks > 1) launch(dev_, stream, local_[vec], blocks, threads_, args, op);
    launch(dev_, stream, forward_[vec], blocks, threads_, args, op);
}

void ScanPlan::backward(const fg_scan_backward_args& a, hipStream_t stream) {
    const char* op = "scan backward";
    const fg_scan_inputs& in = a.in;
    check_inputs(op, in);
    if (a.grad_z.ptr && !in.z.ptr) invalid("scan backward: grad_z without z");
    fg_scan_kargs g = base(in, back_);
    Arrays all(op, s_.packed ? 1 : s_.sequences, s_.packed ? s_.tokens : s_.length, kBytes[s_.dtype]);
    const int64_t state = 4 * s_.sequences * s_.channels * s_.states;
    g.u = all.rows("u", in.u, s_.channels, false);
    g.delta = all.rows("delta", in.delta, s_.channels, false);
    g.b = all.rows("B", in.b, s_.groups * s_.states, false);
    g.c = all.rows("C", in.c, s_.groups * s_.states, false);
    g.z = all.rows("z", in.z, s_.channels, false, true);
    g.gout = all.rows("grad_out", a.grad_out, s_.channels, false);
    g.gu = all.rows("grad_u", a.grad_u, s_.channels, true, true);
    g.gdelta = all.rows("grad_delta", a.grad_delta, s_.channels, true, true);
    g.gb = all.rows("grad_B", a.grad_b, s_.groups * s_.states, true, true);
    g.gc = all.rows("grad_C", a.grad_c, s_.groups * s_.states, true, true);
    g.gz = all.rows("grad_z", a.grad_z, s_.channels, true, true);
    all.flat("A", in.a, 4 * s_.channels * s_.states, false, false);
    all.flat("D", in.d, 4 * s_.channels, false, true);
    all.flat("delta_bias", in.delta_bias, 4 * s_.channels, false, true);
    all.flat("offsets", in.offsets, 4 * (s_.sequences + 1), false, true);
    all.flat("checkpoints", a.checkpoints, (int64_t)checkpoint_bytes(), false, false);
    all.flat("grad_final", a.grad_final, state, false, true);
    all.flat("grad_initial", a.grad_initial, state, true, true);
    all.flat("grad_A", a.grad_a, 4 * s_.channels * s_.states, true, true);
    all.flat("grad_D", a.grad_d, 4 * s_.channels, true, true);
    all.flat("grad_delta_bias", a.grad_delta_bias, 4 * s_.channels, true, true);
    g.check = (float*)a.checkpoints;
    g.gfinal = a.grad_final;
    g.ginitial = a.grad_initial;
    g.ga = a.grad_a;
    g.gskip = a.grad_d;
    g.gbias = a.grad_delta_bias;
    const uint64_t row = 2ull * s_.groups * s_.states, params = (uint64_t)s_.channels * (s_.states + 2);
    {
        std::lock_guard<std::mutex> lock(mu_);
        if (!part_p_.data() && g.seqs) {
            refuse_capture(op, dev_, stream);
            size_of(op, "workspace", {4, group_blocks_, s_.tokens, (int64_t)row});
            size_of(op, "workspace", {4, (int64_t)params, (int64_t)back_.places});
            allocate(back_);
            part_bc_ = Buffer<float, HipBackend>(dev_, group_blocks_ * (uint64_t)s_.tokens * row);
            part_p_ = Buffer<float, HipBackend>(dev_, params * back_.places);
        }
    }
    g.carry = back_.states.data();
    g.carry_dt = back_.dt.data();
    g.part_bc = part_bc_.data();
    g.part_p = part_p_.data();
    const bool vec = wide(g, {&g.u, &g.delta, &g.z, &g.gout, &g.gu, &g.gdelta, &g.gz}, {&g.b, &g.c});
    void* args[] = {&g};
    const uint64_t blocks = (uint64_t)g.seqs * g.chunks * blocks_;
    if (g.chunks > 1) launch(dev_, stream, back_local_[vec], blocks, threads_, args, op);
    launch(dev_, stream, backward_[vec], blocks, threads_, args, op);
    if ((g.gb.p || g.gc.p) && g.seqs) launch(dev_, stream, reduce_bc_, ceil_div(g.tokens * row, 256), 256, args, op);
    if (g.ga || g.gskip || g.gbias) launch(dev_, stream, reduce_p_, ceil_div(params, 256), 256, args, op);
}

}  // namespace fg
