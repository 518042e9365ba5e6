// ssm_ops.hpp -- host side of the sequence filters (kernels/ssm_conv.hpp,
// kernels/ssm_scan.hpp): argument checks, launch geometry and workspaces of
// the short causal convolution and the selective scan.
//
// The kernels are a code object for each element type, loaded by the first plan
// or one-token call of the type: opening a device, which users of the FFT alone
// do too, would take 6.6 ms longer with all three (8.3 / 14.9 ms for a device
// that was open before).
#pragma once

#include <cstdint>
#include <initializer_list>
#include <memory>
#include <mutex>

#include "device.hpp"
#include "hip_backend.hpp"
#include "kernels/ssm_args.h"

namespace fg {

// The code objects of the three element types and the handles of the kernels
// that need no plan.
class SsmKernels {
public:
    explicit SsmKernels(Device<HipBackend>& dev) : dev_(dev) {}

    HipBackend::KernelHandle get(int dtype, const std::string& name) const;

    void conv_step(const HipBackend::DeviceHandle& dev, const fg_conv_step_args& a, hipStream_t stream) const;
    void scan_step(const HipBackend::DeviceHandle& dev, const fg_scan_step_args& a, hipStream_t stream) const;

private:
    struct Type {
        HipBackend::Module mod;
        HipBackend::KernelHandle conv_step[FG_CONV_MAX_WIDTH + 1][3] = {};  // [width][8, 4, 1 channels]
        HipBackend::KernelHandle scan_step[5][2] = {};  // [log2 of a channel's lanes][any, wide]
    };
    const Type& type(int dtype) const;
    Device<HipBackend>& dev_;
    mutable std::mutex mu_;
    mutable std::unique_ptr<Type> types_[3];
};

class ConvPlan {
public:
    ConvPlan(const HipBackend::DeviceHandle& dev, const SsmKernels& k, const fg_conv_shape& s);
    void info(fg_conv_plan_info* out);
    void forward(const fg_conv_forward_args& a, hipStream_t stream) const;
    void backward(const fg_conv_backward_args& a, hipStream_t stream);

private:
    fg_conv_kargs base(const int32_t* offsets) const;
    HipBackend::DeviceHandle dev_;
    fg_conv_shape s_;
    uint32_t run_for(uint32_t n, uint32_t waves, uint32_t least) const;
    uint32_t forward_run(uint32_t n) const;
    uint32_t backward_run() const;
    HipBackend::KernelHandle forward_[3] = {}, backward_[3] = {}, reduce_;  // [8, 4, 1 channels of a thread]
    std::mutex mu_;
    Buffer<float, HipBackend> part_;
};

class ScanPlan {
public:
    ScanPlan(const HipBackend::DeviceHandle& dev, const SsmKernels& k, const fg_scan_shape& s);
    size_t checkpoint_bytes() const;
    void info(fg_scan_plan_info* out);
    void forward(const fg_scan_forward_args& a, hipStream_t stream) const;
    void backward(const fg_scan_backward_args& a, hipStream_t stream);

private:
    // What the chunks of a pass add to the states that pass through them.
    struct Carry {
        uint32_t chunks = 1, chunk_len = 0;  // of a sequence; tokens of a chunk
        uint64_t places = 0;                 // over all sequences
        Buffer<float, HipBackend> states, dt;
    };
    void cut(Carry& c, uint32_t chunks) const;
    void allocate(Carry& c) const;
    fg_scan_kargs base(const fg_scan_inputs& in, const Carry& c) const;
    void check_inputs(const char* op, const fg_scan_inputs& in) const;
    bool wide(const fg_scan_kargs& g, std::initializer_list<const fg_ssm_view*> channels,
              std::initializer_list<const fg_ssm_view*> states) const;
    uint32_t chunks_for(uint32_t few) const;
    HipBackend::DeviceHandle dev_;
    fg_scan_shape s_;
    uint32_t lane_states_, waves_;  // states of a lane, waves that share a channel's states
    uint32_t segment_, threads_, group_blocks_, blocks_;  // blocks_: workgroups over all channels
    HipBackend::KernelHandle local_[2] = {}, forward_[2] = {}, back_local_[2] = {}, backward_[2] = {};  // [any, wide]
    HipBackend::KernelHandle reduce_bc_, reduce_p_;
    Carry ahead_, back_;  // back_'s buffers from the first backward call on
    std::mutex mu_;
    Buffer<float, HipBackend> part_bc_, part_p_;
};

}  // namespace fg
