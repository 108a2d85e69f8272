// Layout constants and checks of the 8-bit cache, shared by its kernels.
#pragma once

#include <stdint.h>

#include "axs6.h"

namespace axs6 {

constexpr int kKvBlock = AXS6_KV_BLOCK;   // tokens that share a scale

int check_cache(const char* fn, int64_t B, int64_t H, int64_t D, int64_t nb, const void* kc, const float* ks,
                const void* vc, const float* vs);

}  // namespace axs6
