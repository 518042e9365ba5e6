// row_arrays.hpp -- what the host sides of the operators over rows of tokens
// (ssm_ops.cpp, rec_ops.cpp, norm_ops.cpp) share: element types, checks of a call's
// sizes and arrays, and launches.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "device.hpp"
#include "hip_backend.hpp"
#include "kernels/ssm_args.h"

namespace fg {
namespace rows {

inline const char* const kTypes[3] = {"f32", "bf16", "f16"};
inline const uint32_t kBytes[3] = {4, 2, 2};
constexpr int64_t kMaxRowStride = 1 << 25;   // 32-bit offsets within a segment's rows
constexpr int64_t kMaxCount = 0x7fffffff;
constexpr int64_t kMaxBytes = int64_t(1) << 46;

inline void check_dtype(const char* op, int64_t dtype) {
    if (dtype < 0 || dtype > 2)
        invalid(std::string(op) + ": dtype must be FG_DTYPE_F32, FG_DTYPE_BF16 or FG_DTYPE_F16, got " +
                std::to_string(dtype));
}

inline void check_range(const char* op, const char* what, int64_t v, int64_t lo, int64_t hi) {
    if (v < lo || v > hi)
        invalid(std::string(op) + ": " + what + " must be in [" + std::to_string(lo) + ", " + std::to_string(hi) +
                "], got " + std::to_string(v));
}

// The product of an array's sizes, refused where no memory holds as many bytes.
inline int64_t size_of(const char* op, const char* what, std::initializer_list<int64_t> sizes) {
    int64_t n = 1;
    for (int64_t k : sizes) {
        if (k > 0 && n > kMaxBytes / k) invalid(std::string(op) + ": " + what + ": too large");
        n *= k;
    }
    return n;
}

// The extent of an array of rows, in bytes from its first element.
struct Extent {
    const char* name = nullptr;
    const char* p = nullptr;
    int64_t bytes = 0;              // up to its last element
    int64_t seq = 0, row = 0;       // bytes
    int64_t width = 0;              // bytes of a row
    bool out = false;
};

// A call's arrays: each is checked when it is added, outputs also against
// everything that was added before and after.
class Arrays {
public:
    Arrays(const char* op, int64_t seqs, int64_t rows, uint32_t es) : op_(op), seqs_(seqs), rows_(rows), es_(es) {}

    // es: bytes of this array's elements where they are not the call's.
    fg_ssm_view rows(const char* name, const fg_rows& r, int64_t width, bool out, bool optional = false, uint32_t es = 0) {
        if (!es) es = es_;
        fg_ssm_view v{nullptr, 0, 0};
        if (!r.ptr) {
            if (!optional && seqs_ > 0 && rows_ > 0) invalid(std::string(op_) + ": " + name + ": null buffer");
            return v;
        }
        v.p = r.ptr;
        v.seq = seqs_ > 1 ? r.seq_stride : 0;
        v.row = rows_ > 1 ? r.row_stride : 0;
        if (reinterpret_cast<uintptr_t>(r.ptr) % es)
            invalid(std::string(op_) + ": " + name + ": not aligned to its elements");
        if (v.seq < 0 || v.row < 0) invalid(std::string(op_) + ": " + name + ": negative stride");
        if (v.row > kMaxRowStride)
            invalid(std::string(op_) + ": " + name + ": row stride " + std::to_string(v.row) + " exceeds " +
                    std::to_string(kMaxRowStride));
        if (seqs_ == 0 || rows_ == 0) return v;
        const __int128 last = (__int128)(seqs_ - 1) * v.seq + (__int128)(rows_ - 1) * v.row + width;
        if (last > kMaxBytes / es) invalid(std::string(op_) + ": " + name + ": too large");
        if (out) {
            // rows of all sequences apart: the larger stride steps over all that the smaller one covers
            int64_t small = v.row, small_n = rows_, large = v.seq, large_n = seqs_;
            if (small_n == 1 || (large_n > 1 && large < small)) std::swap(small, large), std::swap(small_n, large_n);
            if ((small_n > 1 && small < width) || (large_n > 1 && large < (small_n - 1) * small + width))
                invalid(std::string(op_) + ": " + name + ": rows of an output overlap");
        }
        Extent e;
        e.name = name;
        e.p = (const char*)r.ptr;
        e.seq = v.seq * es;
        e.row = v.row * es;
        e.width = width * es;
        e.bytes = (seqs_ - 1) * e.seq + (rows_ - 1) * e.row + e.width;
        e.out = out;
        add(e);
        return v;
    }
    void flat(const char* name, const void* p, int64_t bytes, bool out, bool optional, uint32_t align = 4) {
        if (!p) {
            if (!optional && bytes > 0) invalid(std::string(op_) + ": " + name + ": null buffer");
            return;
        }
        if (reinterpret_cast<uintptr_t>(p) % align)
            invalid(std::string(op_) + ": " + name + ": not aligned to its elements");
        if (bytes <= 0) return;
        Extent e;
        e.name = name;
        e.p = (const char*)p;
        e.bytes = e.width = bytes;
        e.out = out;
        add(e);
    }

private:
    static bool apart(const Extent& a, const Extent& b) {
        if (a.p + a.bytes <= b.p || b.p + b.bytes <= a.p) return true;
        // column windows of one array, whichever of its axes comes first: the same
        // strides, the larger a multiple of the smaller one, and the windows apart within that
        const int64_t least = std::min(a.row, a.seq), most = std::max(a.row, a.seq), step = least > 0 ? least : most;
        if (step <= 0 || a.row != b.row || a.seq != b.seq || most % step) return false;
        int64_t off = (b.p - a.p) % step;
        if (off < 0) off += step;
        return off >= a.width && off + b.width <= step;
    }
    void add(const Extent& e) {
        for (int i = 0; i < n_; ++i) {
            const Extent& x = all_[i];
            if ((e.out || x.out) && !apart(e, x)) invalid(std::string(op_) + ": " + x.name + " and " + e.name + " overlap");
        }
        if (n_ == kMost) fail(FG_ERR_INTERNAL, "more arrays than a call has");
        all_[n_++] = e;
    }
    static constexpr int kMost = 32;  // a call has at most 25
    const char* op_;
    int64_t seqs_, rows_;
    uint32_t es_;
    Extent all_[kMost];
    int n_ = 0;
};

inline void refuse_capture(const char* op, const HipBackend::DeviceHandle& dev, hipStream_t stream) {
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    HipBackend::bind(dev);
    hip_check(hipStreamIsCapturing(HipBackend::stream_of(dev, stream), &cap), "hipStreamIsCapturing");
    if (cap != hipStreamCaptureStatusNone)
        invalid(std::string(op) + ": a plan's first backward call allocates its workspace and cannot be captured");
}

// Device pointers and strides of `v` multiples of a vector of n elements.
inline bool vector_rows(const fg_ssm_view& v, uint32_t n, uint32_t es) {
    return reinterpret_cast<uintptr_t>(v.p) % (n * es) == 0 && v.seq % n == 0 && v.row % n == 0;
}
inline bool vector_ptr(const void* p, uint32_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline void launch(const HipBackend::DeviceHandle& dev, hipStream_t stream, HipBackend::KernelHandle k, uint64_t blocks,
            uint32_t threads, void** args, const char* op) {
    if (blocks == 0) return;
    if (blocks > 0xffffffffull / threads) invalid(std::string(op) + ": too large for one launch");
    HipBackend::launch(dev, stream, k, Dim3((uint32_t)blocks), Dim3(threads), 0, args);
}

inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// A call that is being captured may be the first of its type: loading a code
// object is no work of the stream's, and the thread's capture mode allows it meanwhile.
class CaptureAllows {
public:
    CaptureAllows() { hip_check(hipThreadExchangeStreamCaptureMode(&mode_), "hipThreadExchangeStreamCaptureMode"); }
    ~CaptureAllows() { (void)hipThreadExchangeStreamCaptureMode(&mode_); }

private:
    hipStreamCaptureMode mode_ = hipStreamCaptureModeRelaxed;
};

// Shared by the plans' constructors: sequences, length, tokens.
inline void check_sequences(const char* op, int64_t sequences, int64_t length, int64_t tokens, int64_t packed) {
    check_range(op, "sequences", sequences, 0, kMaxCount);
    check_range(op, "length", length, 0, kMaxCount);
    if (packed) check_range(op, "tokens", tokens, 0, int64_t(1) << 40);
}

// Rows of `width` elements: what is worked out from their number (launches,
// workspaces, checkpoints) stays within 64 bits, also for inputs whose stride of
// 0 lets a small array stand for any number of rows.
template <class Shape>
void check_rows(const char* op, const Shape& s, int64_t width) {
    if (s.packed) size_of(op, "rows", {s.tokens, width, kBytes[s.dtype]});
    else size_of(op, "rows", {s.sequences, s.length, width, kBytes[s.dtype]});
}

}  // namespace rows
}  // namespace fg
