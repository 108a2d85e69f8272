// Device building blocks of the attentions over the 8-bit cache: codes as f16, the
// 16x16x32 products, a row's queries.
#pragma once

#include <math.h>

#include <type_traits>

#include "axs6_internal.h"
#include "kv_cache.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kProbScale = 16384.0f;   // 2^14
constexpr float kSumScale = 1048576.0f;  // 2^20: sums are held as 2^-20 of themselves, so that values near
                                         // float32's largest, summed before they are divided, stay finite

// Eight int8 codes as f16: with the sign bit flipped a byte u is code + 128,
// and the f16 with the bits 0x6400 | u is 1024 + u.  SMALL: times 2^-20 (bits 0x1400 | u),
// 1 / kSumScale, where a block's scale times that might itself be too small for float32.
template <bool SMALL>
__device__ __forceinline__ f16x8 codes_f16(uint32_t a, uint32_t b) {
    constexpr uint32_t kHigh = SMALL ? 0x14141414u : 0x64646464u;
    union { uint32_t w[4]; f16x2 h[4]; f16x8 v; } r;
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    r.w[0] = __builtin_amdgcn_perm(kHigh, a, 0x04010400u);
    r.w[1] = __builtin_amdgcn_perm(kHigh, a, 0x04030402u);
    r.w[2] = __builtin_amdgcn_perm(kHigh, b, 0x04010400u);
    r.w[3] = __builtin_amdgcn_perm(kHigh, b, 0x04030402u);
    constexpr float kBias = SMALL ? 1152.0f / kSumScale : 1152.0f;
    const f16x2 bias = {(_Float16)kBias, (_Float16)kBias};
#pragma unroll
    for (int i = 0; i < 4; ++i) r.h[i] = r.h[i] - bias;
    return r.v;
}

__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// N values of a query from element i.
template <int DT, int N>
__device__ __forceinline__ void load_values(const void* p, int64_t i, bool vec, float* f) {
    using E = Elem<DT>;
    const auto* q = reinterpret_cast<const typename E::S*>(p) + i;
    if (vec) {
#pragma unroll
        for (int j = 0; j < N; j += E::V) E::unpack(*reinterpret_cast<const u32x4*>(q + j), f + j);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = E::to_f(q[j]);
    }
}

// Call f with the dtype code as a constant.
template <class F>
void by_dtype(int dtype, F f) {
    if (dtype == AXS6_F32) f(std::integral_constant<int, AXS6_F32>{});
    else if (dtype == AXS6_BF16) f(std::integral_constant<int, AXS6_BF16>{});
    else f(std::integral_constant<int, AXS6_F16>{});
}

}  // namespace
}  // namespace axs6
