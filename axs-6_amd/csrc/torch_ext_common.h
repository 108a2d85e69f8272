// What the translation units of the torch extension share: dtype codes, the
// current stream, device and status checks.
#pragma once

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>

#include "axs6.h"

namespace axs6_ext {

inline int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return AXS6_F32;
        case at::kBFloat16: return AXS6_BF16;
        case at::kHalf: return AXS6_F16;
        default: return -1;
    }
}

inline void check_rc(int rc, const char* fn) {
    TORCH_CHECK(rc == 0, fn, " failed (status ", rc, "): ", axs6_last_error());
}

inline void require_device(const at::Tensor& t, const char* fn) {
    TORCH_CHECK(t.is_cuda(), fn, " requires a CUDA (ROCm/HIP) device tensor, got device ", t.device());
}

inline void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Row lengths the kernels take without a copy: whole 16-byte vectors (4
// float32 or 8 bfloat16 / float16 values).
inline int64_t vec_multiple(at::ScalarType dtype) { return dtype == at::kFloat ? 4 : 8; }

// The decoder's operators (torch_ext_decoder.cpp).
void register_decoder(py::module& m);

}  // namespace axs6_ext
