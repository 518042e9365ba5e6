// norm_ops.hpp -- host side of the residual norm and of dropout
// (kernels/norm_rows.hpp): argument checks, launch geometry and workspaces.  The
// kernels are a code object for each element type, loaded by the first call of the
// type.
#pragma once

#include <memory>
#include <mutex>

#include "device.hpp"
#include "hip_backend.hpp"
#include "kernels/norm_args.h"

namespace fg {

class NormKernels {
public:
    explicit NormKernels(Device<HipBackend>& dev) : dev_(dev) {}
    HipBackend::KernelHandle get(int dtype, const std::string& name) const;
    void dropout(const HipBackend::DeviceHandle& dev, const fg_dropout_args& a, hipStream_t stream) const;

private:
    struct Type {
        HipBackend::Module mod;
        HipBackend::KernelHandle dropout;
    };
    const Type& type(int dtype) const;
    Device<HipBackend>& dev_;
    mutable std::mutex mu_;
    mutable std::unique_ptr<Type> types_[3];
};

class NormPlan {
public:
    NormPlan(const HipBackend::DeviceHandle& dev, const NormKernels& k, const fg_norm_shape& s);
    void info(fg_norm_plan_info* out);
    void forward(const fg_norm_forward_args& a, hipStream_t stream) const;
    void backward(const fg_norm_backward_args& a, hipStream_t stream);

private:
    uint32_t teams() const;  // of a workgroup
    uint64_t workgroups(uint64_t rows) const;
    fg_norm_kargs base(const char* op, int64_t rows, const float* weight, double dropout, uint64_t seed,
                       uint64_t offset, const int64_t* counter) const;
    HipBackend::DeviceHandle dev_;
    fg_norm_shape s_;
    uint32_t team_;  // threads of a row
    HipBackend::KernelHandle forward_, backward_, reduce_;
    std::mutex mu_;
    Buffer<float, HipBackend> part_;
};

}  // namespace fg
