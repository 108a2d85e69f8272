// The 8-bit cache of keys and values: new tokens in, stored values out.
//
// Tokens stand in blocks of 32.  For a block's tokens that are present, of one
// head, x = key or value values [32][D]:
//   scale = max |x| / 127,  code = round(x / scale) in [-127, 127]  (0 where scale is 0),
// and the block stands for code * scale.  A block with a NaN or infinity gets a
// NaN scale.  Key codes lie as [32][D] (a score reads a token's row), value
// codes as [D][32] (an output value reads one of its tokens' columns), so
// attention's matrix instructions take both without a transposition.
// The block that is not full yet is held raw beside its codes ("tail") and is
// quantized anew from the raw values whenever a token joins it: a block's codes
// depend on its tokens alone, not on the calls that brought them.
//
// Bound by HBM: every value is read once and its code written once; a single
// token's call also reads its block's raw values.
// Measured: 4 x 8191 tokens, 8 heads of 128, bf16, 132 us, 4.1 TB/s (a copy of 4
// GiB runs at 4.7 on this card); 64 sequences' next token 20 to 24 us, the host's
// calls and the launch for the most part.
#include <math.h>

#include "axs6_internal.h"
#include "kv_cache.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kMaxHead = AXS6_KV_MAX_HEAD;
constexpr int kVecs = kKvBlock * kMaxHead / 8 / kAppendThreads;   // 8-value pieces of a block a thread holds

struct AppendArgs {
    const void* x[2];          // keys, values
    int64_t strides[2][3];     // batch, token, head, in elements
    const int64_t* starts;
    int8_t* codes[2];
    float* scales[2];
    void* tail[2];
    int64_t n;
    int H, D, nb;
    int vec[2];                // rows of x are aligned 16-byte vectors
};

// Eight consecutive values as floats; as raw storage for the tail.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, bool vec, float* f) {
    using E = Elem<DT>;
    const auto* q = reinterpret_cast<const typename E::S*>(p) + i;
    if (vec) {
#pragma unroll
        for (int j = 0; j < 8; j += E::V) E::unpack(*reinterpret_cast<const u32x4*>(q + j), f + j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = E::to_f(q[j]);
    }
}
// The floats came from values of the type, so the conversion back is exact.
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* f) {
    using E = Elem<DT>;
    auto* q = reinterpret_cast<typename E::S*>(p) + i;
#pragma unroll
    for (int j = 0; j < 8; j += E::V) *reinterpret_cast<u32x4*>(q + j) = E::pack(f + j);
}

// One workgroup a (sequence, head, touched block, keys or values).
template <int DT>
__global__ __launch_bounds__(kAppendThreads) void kv_append_kernel(AppendArgs a) {
    __shared__ float red[kAppendThreads / 64];
    __shared__ int8_t tile[kKvBlock * (kMaxHead + 4)];
    const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, z = blockIdx.z;
    const int64_t start = a.starts[b], cap = (int64_t)a.nb * kKvBlock;
    if (start < 0 || start >= cap) return;
    const int64_t end = start + a.n < cap ? start + a.n : cap;
    const int64_t blk = start / kKvBlock + blockIdx.y;
    if (blk * kKvBlock >= end) return;
    const int at = blockIdx.y == 0 ? (int)(start % kKvBlock) : 0;            // first new place of the block
    const int to = (int)(end - blk * kKvBlock < kKvBlock ? end - blk * kKvBlock : kKvBlock);
    const int D = a.D, dv = D / 8, pieces = kKvBlock * dv;
    const void* x = a.x[z];
    const int64_t* st = a.strides[z];
    void* tail = a.tail[z];
    const int64_t bh = (int64_t)b * a.H + h, tail0 = bh * kKvBlock * D;
    const int64_t row0 = b * st[0] + h * st[2] + (blk * kKvBlock - start) * st[1];   // place 0 of the block
    float v[kVecs][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = threadIdx.x + i * kAppendThreads, t = c / dv, d = (c - t * dv) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (c < pieces) {
            if (t < at) load8<DT>(tail, tail0 + t * D + d, true, v[i]);
            else if (t < to) load8<DT>(x, row0 + t * st[1] + d, a.vec[z], v[i]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float m = fabsf(v[i][j]);
            amax = m > amax || m != m ? m : amax;   // a NaN stays
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float m = __shfl_xor(amax, o, 64);
        amax = m > amax || m != m ? m : amax;
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();   // and every read of the tail is done
    amax = red[0];
#pragma unroll
    for (int i = 1; i < kAppendThreads / 64; ++i) amax = red[i] > amax || red[i] != red[i] ? red[i] : amax;
    const float scale = isfinite(amax) ? amax / 127.0f : __uint_as_float(0x7fc00000u);
    const bool live = scale > 0.0f;
    const int64_t cell = bh * a.nb + blk, codes0 = cell * kKvBlock * D;
    if (threadIdx.x == 0) a.scales[z][cell] = scale;
    const bool partial = to < kKvBlock;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = threadIdx.x + i * kAppendThreads, t = c / dv, d = (c - t * dv) * 8;
        if (c >= pieces) break;
        uint32_t w[2] = {0, 0};
        if (live) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int q = (int)fminf(fmaxf(rintf(v[i][j] / scale), -127.0f), 127.0f);
                w[j >> 2] |= (uint32_t)(q & 0xff) << (8 * (j & 3));
            }
        }
        if (z == 0) {
            *reinterpret_cast<uint2*>(a.codes[0] + codes0 + t * D + d) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(tile + t * (D + 4) + d) = w[0];
            *reinterpret_cast<uint32_t*>(tile + t * (D + 4) + d + 4) = w[1];
        }
        if (partial && blockIdx.y == 0 && t >= at && t < to) store8<DT>(tail, tail0 + t * D + d, v[i]);
    }
    // The raw values of a partial last block that is not the first one touched
    // are written here too: this workgroup alone reads the tail, and has.
    const int64_t last = end / kKvBlock * kKvBlock;
    if (blockIdx.y == 0 && last > start) {
        const int64_t row = row0 + (last - blk * kKvBlock) * st[1];
        for (int c = threadIdx.x; c < (int)(end - last) * dv; c += kAppendThreads) {
            const int t = c / dv, d = (c - t * dv) * 8;
            float f[8];
            load8<DT>(x, row + t * st[1] + d, a.vec[z], f);
            store8<DT>(tail, tail0 + t * D + d, f);
        }
    }
    if (z == 1) {
        __syncthreads();
        // row d of the codes: its 32 tokens, four to a word
        for (int c = threadIdx.x; c < D * (kKvBlock / 4); c += kAppendThreads) {
            const int d = c / (kKvBlock / 4), t = c % (kKvBlock / 4) * 4;
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) w |= (uint32_t)(uint8_t)tile[(t + j) * (D + 4) + d] << (8 * j);
            *reinterpret_cast<uint32_t*>(a.codes[1] + codes0 + d * kKvBlock + t) = w;
        }
    }
}

struct ReadArgs {
    const int8_t* codes[2];
    const float* scales[2];
    const int64_t* first;
    float* out[2];
    int64_t count;
    int H, D, nb;
};

// One workgroup a (sequence, head, block, keys or values) of the tokens from
// first[b] on; places outside the cache give 0 and nothing is read for them (a cache
// without blocks has no memory).
__global__ __launch_bounds__(kAppendThreads) void kv_read_kernel(ReadArgs a) {
    __shared__ int8_t tile[kMaxHead * (kKvBlock + 4)];
    const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, z = blockIdx.z, D = a.D;
    const int64_t first = a.first[b];
    // the floor of first / 32, also below zero
    const int64_t blk = (first >= 0 ? first / kKvBlock : -((-first + kKvBlock - 1) / kKvBlock)) + blockIdx.y;
    if (blk * kKvBlock >= first + a.count) return;
    const bool inside = blk >= 0 && blk < a.nb;
    const int64_t cell = ((int64_t)b * a.H + h) * a.nb + blk;
    const int8_t* codes = inside ? a.codes[z] + cell * kKvBlock * D : nullptr;
    const float scale = inside ? a.scales[z][cell] : 0.0f;
    if (z == 1 && inside) {
        for (int c = threadIdx.x; c < D * (kKvBlock / 4); c += kAppendThreads) {
            const int d = c / (kKvBlock / 4), t = c % (kKvBlock / 4) * 4;
            *reinterpret_cast<uint32_t*>(tile + d * (kKvBlock + 4) + t) =
                *reinterpret_cast<const uint32_t*>(codes + d * kKvBlock + t);
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < kKvBlock * (D / 4); c += kAppendThreads) {
        const int t = c / (D / 4), d = c % (D / 4) * 4;
        const int64_t i = blk * kKvBlock + t - first;   // place in the output
        if (i < 0 || i >= a.count) continue;
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (inside) {
            uint32_t w = 0;
            if (z == 0) {
                w = *reinterpret_cast<const uint32_t*>(codes + t * D + d);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) w |= (uint32_t)(uint8_t)tile[(d + j) * (kKvBlock + 4) + t] << (8 * j);
            }
            f.x = scale * (float)(int8_t)w;
            f.y = scale * (float)(int8_t)(w >> 8);
            f.z = scale * (float)(int8_t)(w >> 16);
            f.w = scale * (float)(int8_t)(w >> 24);
        }
        *reinterpret_cast<float4*>(a.out[z] + (((int64_t)b * a.count + i) * a.H + h) * D + d) = f;
    }
}

template <int DT>
void launch_append(const AppendArgs& a, int64_t B, int64_t blocks, hipStream_t st) {
    kv_append_kernel<DT><<<dim3((unsigned)(B * a.H), (unsigned)blocks, 2), kAppendThreads, 0, st>>>(a);
}

}  // namespace

int check_cache(const char* fn, int64_t B, int64_t H, int64_t D, int64_t nb, const void* kc, const float* ks,
                const void* vc, const float* vs) {
    if (B < 0 || H < 0 || nb < 0) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: negative dimension", fn);
    if (D <= 0 || D % 16 || D > kMaxHead)
        return fail(AXS6_ERR_UNSUPPORTED, "%s: heads of a multiple of 16 values up to %d, got %lld", fn, kMaxHead,
                    (long long)D);
    if (B * H > ((int64_t)1 << 31) - 1 || nb > ((int64_t)1 << 25))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    if (B * H * nb == 0) return AXS6_OK;
    if (!kc || !ks || !vc || !vs) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
    if ((uintptr_t)kc % 16 || (uintptr_t)vc % 16 || (uintptr_t)ks % 4 || (uintptr_t)vs % 4)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: codes not aligned to 16 bytes, or scales to 4", fn);
    return AXS6_OK;
}

}  // namespace axs6

using namespace axs6;

extern "C" int axs6_kv_append(const void* k, const void* v, int32_t dtype, int64_t B, int64_t n, int64_t H, int64_t D,
                              const int64_t* k_strides, const int64_t* v_strides, const int64_t* starts,
                              int64_t blocks, void* k_codes, float* k_scales, void* v_codes, float* v_scales,
                              void* k_tail, void* v_tail, void* stream) {
    const char* fn = "axs6_kv_append";
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    int rc = check_cache(fn, B, H, D, blocks, k_codes, k_scales, v_codes, v_scales);
    if (rc) return rc;
    if (n < 0 || n > ((int64_t)1 << 31)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: bad number of tokens", fn);
    if (n == 0 || B * H * blocks == 0) return AXS6_OK;
    if (!k || !v || !k_strides || !v_strides || !starts || !k_tail || !v_tail)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null keys, values, strides, starts or tail", fn);
    const int64_t es = dtype == AXS6_F32 ? 4 : 2, vl = 16 / es;
    if ((uintptr_t)k % es || (uintptr_t)v % es || (uintptr_t)k_tail % 16 || (uintptr_t)v_tail % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not aligned", fn);
    AppendArgs a{};
    a.x[0] = k; a.x[1] = v; a.starts = starts;
    a.codes[0] = reinterpret_cast<int8_t*>(k_codes); a.codes[1] = reinterpret_cast<int8_t*>(v_codes);
    a.scales[0] = k_scales; a.scales[1] = v_scales; a.tail[0] = k_tail; a.tail[1] = v_tail;
    a.n = n; a.H = (int)H; a.D = (int)D; a.nb = (int)blocks;
    a.vec[0] = (uintptr_t)k % 16 == 0; a.vec[1] = (uintptr_t)v % 16 == 0;
    for (int i = 0; i < 3; ++i) {
        a.strides[0][i] = k_strides[i]; a.strides[1][i] = v_strides[i];
        a.vec[0] = a.vec[0] && k_strides[i] % vl == 0;
        a.vec[1] = a.vec[1] && v_strides[i] % vl == 0;
    }
    // blocks that n tokens touch at most, from any place of the first
    int64_t touched = (n + kKvBlock - 2) / kKvBlock + 1;
    if (touched > blocks) touched = blocks;
    if (touched > 65535) return fail(AXS6_ERR_UNSUPPORTED, "%s: at most %d tokens a call", fn, 65534 * kKvBlock);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AXS6_F32) launch_append<AXS6_F32>(a, B, touched, st);
    else if (dtype == AXS6_BF16) launch_append<AXS6_BF16>(a, B, touched, st);
    else launch_append<AXS6_F16>(a, B, touched, st);
    return check_launch(fn);
}

extern "C" int axs6_kv_read(const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales,
                            int64_t B, int64_t H, int64_t D, int64_t blocks, const int64_t* first, int64_t count,
                            float* k_out, float* v_out, void* stream) {
    const char* fn = "axs6_kv_read";
    int rc = check_cache(fn, B, H, D, blocks, k_codes, k_scales, v_codes, v_scales);
    if (rc) return rc;
    if (count < 0 || count > (int64_t)65534 * kKvBlock)
        return fail(AXS6_ERR_UNSUPPORTED, "%s: 0 to %d tokens a call", fn, 65534 * kKvBlock);
    if (B * H * count == 0) return AXS6_OK;
    if (!first || !k_out || !v_out || (uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null first, or output null or not aligned to 16 bytes", fn);
    ReadArgs a{};
    a.codes[0] = reinterpret_cast<const int8_t*>(k_codes); a.codes[1] = reinterpret_cast<const int8_t*>(v_codes);
    a.scales[0] = k_scales; a.scales[1] = v_scales; a.first = first; a.out[0] = k_out; a.out[1] = v_out;
    a.count = count; a.H = (int)H; a.D = (int)D; a.nb = (int)blocks;
    const int64_t touched = (count + kKvBlock - 2) / kKvBlock + 1;
    kv_read_kernel<<<dim3((unsigned)(B * H), (unsigned)touched, 2), kAppendThreads, 0, (hipStream_t)stream>>>(a);
    return check_launch(fn);
}
