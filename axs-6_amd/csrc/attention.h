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
//   float32: 32x32x2, columns by 4-byte reads, those of all the row's results at once.
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
    float2* stats;                     // (B, Hq, Tq): row_stats
    float* delta;                      // (B, Hq, Tq)
    float2* bounds;                    // (B, Hq, Tq / 32 rounded up): 32 queries' largest |do| and |delta| (float16)
    // Splits of the walked axis and their partial results: of the forward each
    // row's sums, maximum and sum; of the backward dq, and dk and dv.
    int splits, splits_kv;
    float *part, *stat, *part_kv;
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

// Rows of DC values (a multiple of 16) at a pitch of 64 or 128 values; the
// 16-byte chunk c of a row lies in slot c ^ key(row).  gfx950's LDS serves 256
// bytes at once: the key spreads a fragment's 16 rows over all of them, and
// the four rows (16-bit) or two rows (float32) of a column read as well.
template <int DT, int DC>
struct Tile {
    static_assert(DC % 16 == 0 && DC <= 128, "a multiple of a product's depth");
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

    // Column 32 d + l % 32 of the 16 rows from row0 (16-bit types).
    __device__ static u32x4 col_fragment(const char* tile, int row0, int d, int lane) {
        const int h = lane >> 5, s = lane & 15, chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
        u32x4 a;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = row0 + 8 * e + 4 * h + (s >> 2);
            const s16x4 x =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + at(row, chunk) + (s & 1) * 8));
            const u32x2 w = __builtin_bit_cast(u32x2, x);
            a[2 * e] = w[0];
            a[2 * e + 1] = w[1];
        }
        return a;
    }

    // Results over a tile's columns: DC / 32 of them, rounded up.  Row r of result d is
    // column 32 d + r of the tile in the 16-bit types.  In float32 a lane reads
    // the columns of several results at once: column 4 r + d of four, 2 r + d of
    // the first two, 64 + r of the third of three.
    static constexpr int kResults = (DC + 31) / 32;

    // o += (the 32 rows from row0)^T p, p a result whose rows are these rows; pf: p
    // in fragments (16-bit types).
    __device__ static void accumulate(const char* tile, int row0, const f32x16& p, const u32x4 (&pf)[2],
                                      f32x16 (&o)[kResults], int lane) {
        if constexpr (DT == AXS6_F32) {
            const int m = lane & 31;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = row0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
                float x[4];
                if constexpr (kResults == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(tile + at(row, m));
                    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(tile + at(row, m >> 1) + (m & 1) * 8);
                    x[0] = v.x; x[1] = v.y;
                    if constexpr (kResults == 3)
                        x[2] = *reinterpret_cast<const float*>(tile + at(row, 16 + (m >> 2)) + (m & 3) * 4);
                }
#pragma unroll
                for (int d = 0; d < kResults; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[d], p[i], o[d], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int d = 0; d < kResults; ++d)
#pragma unroll
                for (int j = 0; j < 2; ++j) o[d] = mma<DT>(col_fragment(tile, row0 + 16 * j, d, lane), pf[j], o[d]);
        }
    }

    // The results, times f, as the lane's row of memory (element `row` of out) in
    // the type OUT.
    template <int OUT>
    __device__ static void store(void* out, int64_t row, const f32x16 (&o)[kResults], float f, int D, int lane) {
        auto* p = reinterpret_cast<typename Elem<OUT>::S*>(out) + row;
        const int h4 = 4 * (lane >> 5);
        if constexpr (DT == AXS6_F32) {
            static_assert(OUT == AXS6_F32, "float32 results");
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 8 * (i >> 2) + h4 + (i & 3);
                if constexpr (kResults == 4) {
                    if (4 * r < D)
                        *reinterpret_cast<float4*>(p + 4 * r) =
                            make_float4(o[0][i] * f, o[1][i] * f, o[2][i] * f, o[3][i] * f);
                } else {
                    if (2 * r < D) *reinterpret_cast<float2*>(p + 2 * r) = make_float2(o[0][i] * f, o[1][i] * f);
                    if constexpr (kResults == 3)
                        if (64 + r < D) p[64 + r] = o[2][i] * f;
                }
            }
        } else {
#pragma unroll
            for (int d = 0; d < kResults; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int col = 32 * d + 8 * g + h4;
                    const float x = o[d][4 * g] * f, y = o[d][4 * g + 1] * f, z = o[d][4 * g + 2] * f,
                                w = o[d][4 * g + 3] * f;
                    if (col >= D) continue;
                    if constexpr (OUT == AXS6_F32) *reinterpret_cast<float4*>(p + col) = make_float4(x, y, z, w);
                    else *reinterpret_cast<uint2*>(p + col) = make_uint2(pack2<OUT>(x, y), pack2<OUT>(z, w));
                }
        }
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

// The buffer descriptor of `bytes` bytes from p: loads past it give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
    const int n = bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : (int)bytes;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, n, 0x00020000);
}
typedef __attribute__((address_space(3))) void lds_void;

// A tile of R rows straight from memory into LDS (16 bytes a lane, 1 KB a wave
// and instruction, in slot order): values past D arrive as zeros, and so do rows
// past the last one where rows lie a row's bytes apart or more; of rows that overlap
// (an expanded dim) some are real values, so what multiplies them has to be 0.  The
// caller waits on vmcnt and a barrier.
template <int DT, int DC, int R, int WAVES>
struct Direct {
    using T = Tile<DT, DC>;
    static constexpr int kSlots = T::kPitch / 16, kN = R * kSlots / 64 / WAVES;
    static_assert(R * kSlots % (64 * WAVES) == 0, "whole instructions a wave");
    int off[kN];
    int pitch;   // bytes from a row to the next
    __device__ void init(int64_t stride, int D, int lane, int w) {
        pitch = (int)(stride * T::kBytes);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int p = (i * WAVES + w) * 64 + lane, row = p / kSlots, chunk = (p % kSlots) ^ T::key(row);
            off[i] = chunk * T::kVals < D ? row * pitch + chunk * 16 : 0x7fffffff;
        }
    }
    // rows row0 .. row0 + R - 1 of `rows`
    __device__ void load(char* tile, const char* base, int row0, int rows, int D, int w) const {
#if defined(__HIP_DEVICE_COMPILE__)   // the host pass knows no 16-byte form and would drop the kernel's stub
        const int left = rows - row0 < R ? rows - row0 : R;
        const auto rsrc = buffer_of(base + (int64_t)row0 * pitch, left <= 0 ? 0 : (int64_t)(left - 1) * pitch + D * T::kBytes);
#pragma unroll
        for (int i = 0; i < kN; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(tile + (i * WAVES + w) * 1024), 16, off[i], 0, 0, 0);
#endif
    }
};

// Every load of this wave has arrived and every LDS read of it is done, then
// the workgroup meets: tiles on their way may be read, read ones overwritten.
__device__ __forceinline__ void tile_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The head and the piece (of `pieces`, the longest first) that workgroup `id`
// takes.  Consecutive ids go round the 8 XCDs: where the heads divide by 8 each
// XCD takes whole heads, one after another, whose keys its L2 then holds
// (by_piece: all heads' first pieces, then their second ones); else the pieces go
// round all heads, so that every XCD gets long and short ones.
__device__ __forceinline__ void work_item(int id, int heads, int pieces, bool by_piece, int& head, int& piece) {
    if (heads % 8 == 0) {
        const int per = heads / 8, i = id >> 3;
        head = (id & 7) * per + (by_piece ? i % per : i / pieces);
        piece = by_piece ? i / per : i % pieces;
    } else {
        head = id % heads;
        piece = id / heads;
    }
}

// l + the sum of a fragment's values, as they are in the type.
template <int DT>
__device__ __forceinline__ float add_fragment(u32x4 f, float l) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = f[i];
        if constexpr (DT == AXS6_F16) {
            typedef _Float16 x2 __attribute__((ext_vector_type(2)));
            l = __builtin_amdgcn_fdot2(__builtin_bit_cast(x2, x), x2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
        } else {
            typedef __bf16 x2 __attribute__((ext_vector_type(2)));
            l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(x2, x), x2{(__bf16)1.0f, (__bf16)1.0f}, l, false);
        }
    }
    return l;
}

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

// How a mask is read: not at all; by key (the same for all queries of a head: a
// tile's terms lie in LDS); by query and key.  The backward tells masks by key that add
// values from those that only hide: a row's maximum may then be of any size.
enum MaskKind { kNoMask, kKeyMask, kFullMask, kKeyAdd };
constexpr bool by_key(int mask) { return mask == kKeyMask || mask == kKeyAdd; }
constexpr bool adds(int mask) { return mask == kFullMask || mask == kKeyAdd; }

// What a row's probabilities are made from again: p = exp2((x - y) - z), x the score in
// units of log2, for y = m + log2 l and z = 0, or y = m and z = log2 l where float32 has
// no place for log2 l beside m (the keys of a row all carry -1e9, which leaves m there).
// 64: log2 l is then off by 2^-19 at the most, 1.3e-6 of a probability.  A row that sees
// nothing has y = +inf.
__device__ __forceinline__ float2 row_stats(float m, float l) {
    const float s = __builtin_amdgcn_logf(l);
    if (l == 0.0f) return make_float2(INFINITY, 0.0f);
    return fabsf(m) < 64.0f ? make_float2(m + s, 0.0f) : make_float2(m, s);
}

// What the mask adds to a score in units of log2: -inf where the query does not
// see the key.  An added value below -1e38 counts as that: times log2(e) it
// would be -inf, and a row of the type's lowest values, which averages all its
// keys, would be taken for an empty one.
__device__ __forceinline__ float mask_term(const AttnArgs& a, const char* row, int64_t k) {
    if (a.mask_type < 0) return row[k * a.ms[3]] ? 0.0f : -INFINITY;
    const float add = load_elem(row, a.mask_type, k * a.ms[3]);
    return add == -INFINITY || add != add ? add : fmaxf(add, -1e38f) * kLog2e;
}
__device__ __forceinline__ const char* mask_row(const AttnArgs& a, int b, int h, int64_t q) {
    const int64_t bytes = a.mask_type < 0 ? 1 : a.mask_type == AXS6_F32 ? 4 : 2;
    return reinterpret_cast<const char*>(a.mask) + (b * a.ms[0] + h * a.ms[1] + q * a.ms[2]) * bytes;
}
// The terms of the four keys from k (those below Tk): one load where the mask is
// bytes, adjacent and aligned.
__device__ __forceinline__ void mask_terms(const AttnArgs& a, const char* row, int k, float (&f)[4]) {
    const char* p = row + k;
    if (a.mask_type < 0 && a.ms[3] == 1 && k + 4 <= a.Tk && (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = (w >> (8 * e)) & 0xff ? 0.0f : -INFINITY;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = k + e < a.Tk ? mask_term(a, row, k + e) : -INFINITY;
    }
}

// The scores s of 32 keys from k0 (rows of the result) against the lane's
// query: with the mask, in units of log2, unless it is `plain` here; `edge`: keys
// at or past limit are not seen.  term: the keys' terms in LDS (by key).
template <int MASK>
__device__ __forceinline__ void apply_mask(const AttnArgs& a, f32x16& s, float c, int k0, const float* term,
                                           const char* row, bool plain, bool edge, int limit, int lane) {
    const int h4 = 4 * (lane >> 5);
    if (MASK != kNoMask && !plain) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float f[4];
            if constexpr (by_key(MASK)) {
                const float4 t = *reinterpret_cast<const float4*>(term + 8 * g + h4);
                f[0] = t.x; f[1] = t.y; f[2] = t.z; f[3] = t.w;
            } else {
                mask_terms(a, row, k0 + 8 * g + h4, f);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * g + e] = __builtin_fmaf(s[4 * g + e], c, f[e]);
        }
    }
    if (edge)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[i] = k0 + 8 * (i >> 2) + h4 + (i & 3) < limit ? s[i] : -INFINITY;
}

// Adds the second group's results to the first's: the four waves of each group
// hold the same rows.  ex: 4 * N * 16 * 64 floats of LDS that nobody uses; every
// wave of the workgroup calls it.
template <int N>
__device__ __forceinline__ void add_groups(f32x16 (&c)[N], float* ex, int group, int w, int lane) {
    __syncthreads();
    ex += w * (N * 16) * 64 + lane;
    if (group == 1)
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) ex[(16 * d + i) * 64] = c[d][i];
    __syncthreads();
    if (group == 0)
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) c[d][i] += ex[(16 * d + i) * 64];
}

// ---- rows again -------------------------------------------------------------
// A key that a query does not see has no part in its results, whatever key and
// value hold there.  An infinity or NaN there turns the mask's -inf and the weight of 0 in the
// products over a tile's rows into NaN; so a result that is not finite is made
// again from the pairs that see each other alone, one pair at a time by one wave.
// Where those give a NaN everywhere there is nothing more to find.  That is slow, and an
// infinity that is seen costs it too: 1 x 1024, 8 heads on 2 of 64, 16 bit, forward and
// backward 0.12 ms, with one infinity in dout 4.6, in one value 9.5; a wave's 32 rows go
// over all their pairs, so the time grows with the length (and the group's heads).

// Whether any of the results of the lane's column is not finite.
template <int N>
__device__ __forceinline__ bool not_finite(const f32x16 (&c)[N]) {
    float z = 0.0f;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) z = __builtin_fmaf(c[d][i], 0.0f, z);
    z += __shfl_xor(z, 32, 64);
    return z != z;
}

// Values l and l + 64 of a row of D.
struct Two { float x, y; };
template <int DT>
__device__ __forceinline__ Two load_two(const void* p, int64_t i, int D, int lane) {
    using E = Elem<DT>;
    const auto* q = reinterpret_cast<const typename E::S*>(p) + i;
    return {lane < D ? E::to_f(q[lane]) : 0.0f, lane + 64 < D ? E::to_f(q[lane + 64]) : 0.0f};
}
template <int DT>
__device__ __forceinline__ void store_two(void* p, int64_t i, Two v, int D, int lane) {
    using E = Elem<DT>;
    auto* q = reinterpret_cast<typename E::S*>(p) + i;
    if (lane < D) q[lane] = E::from_f(v.x);
    if (lane + 64 < D) q[lane + 64] = E::from_f(v.y);
}
__device__ __forceinline__ float dot(Two a, Two b) {
    float s = a.x * b.x + a.y * b.y;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    return s;
}
__device__ __forceinline__ bool all_nan(Two v, int D, int lane) {
    return __all((lane >= D || v.x != v.x) && (lane + 64 >= D || v.y != v.y));
}
// What the masks add to the score of the pair, -inf where it is not seen.
__device__ __forceinline__ float pair_term(const AttnArgs& a, int b, int hq, int q, int key) {
    if (a.causal && key > q + a.Tk - a.Tq) return -INFINITY;
    return a.mask ? mask_term(a, mask_row(a, b, hq, q), key) : 0.0f;
}

}  // namespace

// Defined in attention_bwd.hip.
int attention_backward(const AttnArgs& a, int dtype, hipStream_t st);

}  // namespace axs6
