// rec_ops.hpp -- host side of the gated linear recurrence (kernels/rec_scan.hpp):
// argument checks, launch geometry and workspaces.  The kernels are a code object
// for each element type, loaded by the first plan or one-token call of the type.
#pragma once

#include <memory>
#include <mutex>

#include "device.hpp"
#include "hip_backend.hpp"
#include "kernels/rec_args.h"

namespace fg {

class RecurrenceKernels {
public:
    explicit RecurrenceKernels(Device<HipBackend>& dev) : dev_(dev) {}
    HipBackend::KernelHandle get(int dtype, const std::string& name) const;
    void step(const HipBackend::DeviceHandle& dev, const fg_recurrence_step_args& a, hipStream_t stream) const;

private:
    struct Type {
        HipBackend::Module mod;
        HipBackend::KernelHandle step[2] = {};  // [any, wide]
    };
    const Type& type(int dtype) const;
    Device<HipBackend>& dev_;
    mutable std::mutex mu_;
    mutable std::unique_ptr<Type> types_[3];
};

class RecurrencePlan {
public:
    RecurrencePlan(const HipBackend::DeviceHandle& dev, const RecurrenceKernels& k, const fg_recurrence_shape& s);
    size_t checkpoint_bytes() const;
    void info(fg_recurrence_plan_info* out);
    void forward(const fg_recurrence_forward_args& a, hipStream_t stream) const;
    void backward(const fg_recurrence_backward_args& a, hipStream_t stream);

private:
    // Of a pass, which has kernels of its own: tokens of a wave, waves of a
    // workgroup, tiles over all chains and channels, and what they pass on.
    uint32_t wave_tokens(bool back) const;
    uint32_t waves(bool back) const;
    uint64_t places(bool back) const;
    Buffer<char, HipBackend> chain(bool back) const;
    fg_rec_kargs base(const char* op, const fg_recurrence_inputs& in, bool back) const;
    HipBackend::DeviceHandle dev_;
    fg_recurrence_shape s_;
    uint64_t chains_, rows_;  // chains of so many rows: dense, the sequences; packed, one
    uint32_t blocks_;         // workgroups over the channels
    HipBackend::KernelHandle forward_[2] = {}, backward_[2] = {}, reduce_;  // [any, wide]
    Buffer<char, HipBackend> ahead_, back_;  // what the tiles pass on, back_ from the first backward call on
    std::mutex mu_;
    Buffer<float, HipBackend> part_;
};

}  // namespace fg
