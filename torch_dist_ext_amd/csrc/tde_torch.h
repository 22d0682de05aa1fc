// What the operator registrations share: status and dtype translation, and the device, stream and outputs of a call.
#ifndef TDE_TORCH_H
#define TDE_TORCH_H

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/hip/HIPContextLight.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include "tde_abi.h"

namespace {

using at::Tensor;

[[maybe_unused]] void check_status(int st, const char *what) {
    if (st == TDE_OK) return;
    if (st == TDE_EHIP) {
        TORCH_CHECK(false, what, ": ", tde_status_string(st), ", hipError ", tde_last_hip_error());
    }
    TORCH_CHECK(false, what, ": ", tde_status_string(st));
}

[[maybe_unused]] int32_t dtype_code(const Tensor &t) {
    switch (t.scalar_type()) {
    case at::kBFloat16: return TDE_BF16;
    case at::kHalf: return TDE_F16;
    case at::kFloat: return TDE_F32;
    case at::kDouble: return TDE_F64;
    default: TORCH_CHECK(false, "torch_dist_ext: unsupported dtype ", t.scalar_type(), " (bf16, fp16, fp32, fp64)");
    }
    return -1;
}

// The device of a call's tensors, made the current one for the call's duration.
class CallDevice {
public:
    explicit CallDevice(const Tensor &on) : index_(on.device().index()) {
        if (index_ != c10::hip::current_device()) guard_.set_index(index_);
    }

    // A new output tensor, straight from the allocator.  at::empty and at::empty_like go through the dispatcher once and twice
    // more, at::detail::empty_cuda asks for the device and the global context each time.  A call's host time without its launch,
    // through both, empty_cuda and this: allreduce_rms 2.14 -> 1.78 us from the second to the third, allreduce_rms_quant 3.15 -> 2.49
    // (from the first to the second 0.2-0.3 us an output).
    Tensor new_output(at::IntArrayRef sizes, at::ScalarType dtype) const {
        return Tensor(at::detail::empty_generic(sizes, allocator_, c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype, c10::nullopt));
    }
    Tensor new_like(const Tensor &t) const { return new_output(t.sizes(), t.scalar_type()); }

    hipStream_t stream() const { return c10::hip::getCurrentHIPStream(index_).stream(); }

private:
    c10::DeviceIndex index_;
    c10::hip::OptionalHIPGuard guard_;
    c10::Allocator *allocator_ = at::cuda::getCUDADeviceAllocator();
};

} // namespace

#endif // TDE_TORCH_H
