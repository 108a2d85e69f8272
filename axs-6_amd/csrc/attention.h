// Device building blocks of attention's forward and backward (gfx950): LDS
// tiles, the 32x32 matrix products on them, masks.
//
// A tile holds rows (queries or keys) of DC values.  Products take it in two
// ways: "rows" (contracted over a row's values, 16 bytes a lane) and "columns"
// (contracted over the tile's rows).  A 32x32 result has in lane l, register i
//   column l % 32, row 8 (i / 4) + 4 (l / 32) + i % 4,
// and the products over the tile's rows take their rows in that same order, so
// a result (probabilities, their gradients) is the next product's operand
// without leaving its registers.
//   16-bit types: 32x32x16, columns by transposing LDS reads of 4 rows;
//   float32: 32x32x2, columns by plain 4-byte reads.
#pragma once

#include <math.h>

#include "axs6_internal.h"
#include "nf5_device.h"

#pragma clang fp contract(fast)

namespace axs6 {

struct AttnArgs {
    const void *q, *k, *v, *out, *dout;
    void *o, *dq, *dk, *dv;            // contiguous (B, T, H, D)
    int64_t qs[3], ks[3], vs[3], os[3], gs[3];   // strides of batch, token, head (q, k, v, out, dout)
    float *lse, *delta;                // (B, Hq, Tq); lse in units of log2, +inf where a row sees nothing
    const void* mask;
    int64_t ms[4];                     // strides of batch, head, query, key
    int mask_type;                     // -1: bytes, true where a query sees a key; else a type code: added
    int B, Hq, H, G, Tq, Tk, D, causal;
    float scale;
};

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f;

template <int DT> constexpr int kElemBytes = DT == AXS6_F32 ? 4 : 2;

// c + A B^T of two fragments of 16 bytes a lane: the lane's row is l % 32, its
// values the half l / 32 of the step's.
template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == AXS6_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    } else if constexpr (DT == AXS6_F16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0,
                                                      0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// Two floats to one word of the type, rounded to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    if constexpr (DT == AXS6_BF16) {
        typedef __bf16 x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, x2));
    } else {
        typedef _Float16 x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, x2));
    }
}

// Rows of DC values (a multiple of 32) at a pitch of 64 or 128 values; the
// 16-byte chunk c of a row lies in slot c ^ key(row).  gfx950's LDS serves 256
// bytes at once: the key spreads a fragment's 16 rows over all of them, and
// the four rows (16-bit) or two rows (float32) of a column read as well.
template <int DT, int DC>
struct Tile {
    static constexpr int kBytes = kElemBytes<DT>;
    static constexpr int kPitch = (DC <= 64 ? 64 : 128) * kBytes;
    static constexpr int kChunks = DC * kBytes / 16;    // of a row
    static constexpr int kSteps = kChunks / 2;          // products over a row
    static constexpr int kVals = 16 / kBytes;           // values of a chunk

    __device__ static int key(int row) {
        if constexpr (DT == AXS6_F32) return ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3);
        else if constexpr (kPitch == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else return ((row & 3) << 2) | ((row >> 2) & 3);
    }
    __device__ static int at(int row, int chunk) { return row * kPitch + ((chunk ^ key(row)) << 4); }

    // Row row0 + l % 32, step s.
    __device__ static u32x4 rows(const char* tile, int row0, int s, int lane) {
        return *reinterpret_cast<const u32x4*>(tile + at(row0 + (lane & 31), 2 * s + (lane >> 5)));
    }

    // c += (columns 32 d .. 32 d + 31 of the 32 rows from row0)^T p, p a result
    // whose rows are these rows; pf: p in fragments (16-bit types).
    __device__ static f32x16 cols(const char* tile, int row0, int d, const f32x16& p, const u32x4 (&pf)[2], f32x16 c,
                                  int lane) {
        const int h = lane >> 5;
        if constexpr (DT == AXS6_F32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = row0 + 8 * (i >> 2) + 4 * h + (i & 3), col = 32 * d + (lane & 31);
                const float x = *reinterpret_cast<const float*>(tile + at(row, col >> 2) + (col & 3) * 4);
                c = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[i], c, 0, 0, 0);
            }
        } else {
            const int s = lane & 15, chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                u32x4 a;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = row0 + 16 * j + 8 * e + 4 * h + (s >> 2);
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)(tile + at(row, chunk) + (s & 1) * 8));
                    const u32x2 w = __builtin_bit_cast(u32x2, x);
                    a[2 * e] = w[0];
                    a[2 * e + 1] = w[1];
                }
                c = mma<DT>(a, pf[j], c);
            }
        }
        return c;
    }
};

// A 32x32 result as the operand of a product over its rows.
template <int DT>
__device__ __forceinline__ void fragments(const f32x16& p, u32x4 (&pf)[2]) {
    if constexpr (DT != AXS6_F32) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) pf[j][e] = pack2<DT>(p[8 * j + 2 * e], p[8 * j + 2 * e + 1]);
    }
}

// A tile of R rows on its way from memory through registers into LDS; rows at
// or past `rows` and values at or past D are zeros.
template <int DT, int DC, int R, int THREADS>
struct Stage {
    using T = Tile<DT, DC>;
    static constexpr int kAll = R * T::kChunks, kN = (kAll + THREADS - 1) / THREADS;
    u32x4 r[kN];
    __device__ void load(const void* base, int64_t stride, int row0, int rows, int D) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = threadIdx.x + i * THREADS, row = c / T::kChunks, ch = c % T::kChunks;
            r[i] = u32x4{0, 0, 0, 0};
            if (c < kAll && row0 + row < rows && ch * T::kVals < D)
                r[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) +
                                                       ((row0 + row) * stride + ch * T::kVals) * T::kBytes);
        }
    }
    __device__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = threadIdx.x + i * THREADS;
            if (kAll % THREADS == 0 || c < kAll)
                *reinterpret_cast<u32x4*>(tile + T::at(c / T::kChunks, c % T::kChunks)) = r[i];
        }
    }
};

// One row of memory as row fragments: the lane's row is l % 32.
template <int DT, int DC, int N>
__device__ __forceinline__ void load_rows(u32x4 (&f)[N], const void* base, int64_t offset, int D, int lane) {
    using T = Tile<DT, DC>;
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const int ch = 2 * s + (lane >> 5);
        f[s] = u32x4{0, 0, 0, 0};
        if (ch * T::kVals < D)
            f[s] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) +
                                                   (offset + ch * T::kVals) * T::kBytes);
    }
}

// What the mask makes of x (the score times scale log2(e)); -inf where the
// query does not see the key.  An added value below -1e38 counts as that: times
// log2(e) it would be -inf, and a row of the type's lowest values, which
// averages all its keys, would be taken for an empty one.
__device__ __forceinline__ float masked(const AttnArgs& a, const char* row, int64_t k, float x) {
    if (a.mask_type < 0) return row[k * a.ms[3]] ? x : -INFINITY;
    const float add = load_elem(row, a.mask_type, k * a.ms[3]);
    return add == -INFINITY ? -INFINITY : x + fmaxf(add, -1e38f) * kLog2e + (add != add ? add : 0.0f);
}
__device__ __forceinline__ const char* mask_row(const AttnArgs& a, int b, int h, int64_t q) {
    const int64_t bytes = a.mask_type < 0 ? 1 : a.mask_type == AXS6_F32 ? 4 : 2;
    return reinterpret_cast<const char*>(a.mask) + (b * a.ms[0] + h * a.ms[1] + q * a.ms[2]) * bytes;
}

// A 32x32 result whose lanes are rows of memory: out[row][32 d + ...] of the
// type, 4 values at a time.
template <int DT>
__device__ __forceinline__ void store_cols(void* out, int64_t row, int d, const f32x16& c, float f, int D, int lane) {
    using E = Elem<DT>;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int col = 32 * d + 8 * g + 4 * (lane >> 5);
        if (col >= D) continue;
        auto* p = reinterpret_cast<typename E::S*>(out) + row + col;
        if constexpr (DT == AXS6_F32) {
            *reinterpret_cast<float4*>(p) = make_float4(c[4 * g] * f, c[4 * g + 1] * f, c[4 * g + 2] * f, c[4 * g + 3] * f);
        } else {
            *reinterpret_cast<uint2*>(p) =
                make_uint2(pack2<DT>(c[4 * g] * f, c[4 * g + 1] * f), pack2<DT>(c[4 * g + 2] * f, c[4 * g + 3] * f));
        }
    }
}

}  // namespace

// Defined in attention_bwd.hip.
int attention_backward(const AttnArgs& a, int dtype, hipStream_t st);

}  // namespace axs6
