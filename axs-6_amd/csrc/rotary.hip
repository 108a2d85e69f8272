// Rotary positions of queries and keys, both layouts, any even part of the
// head, in one launch.
//
// For a token at position p and pair i < R/2 with c = cos, s = sin from the
// table's row p (R/2 cosines, then R/2 sines, float32; any scaling for long
// contexts is in the table):
//   (a, b) = (x[i], x[i + R/2])    half layout
//            (x[2i], x[2i + 1])    interleaved layout
//   (a, b) -> (a c - b s, b c + a s);  x[R..D) is copied.
// The backward is the inverse rotation (s negated): the map is orthogonal up
// to the table's own factor, so its transpose is the same with -s.
//
// Bound by HBM: each value is read once and written once.  A thread keeps the
// cosines and sines of its place in the head in registers and walks over
// heads of one token, so the table is read once a token and not once a head.
// Measured, bf16, 40 heads of 128: 2 x 4096 tokens 28 us, 6.0 TB/s (two
// thirds from the last cache), interleaved 34; 4 x 4095 forward and backward
// 276 us, 4.9 TB/s, a copy's rate from memory; one token 7 us, of which the launch
// is nearly all.
#include "axs6_internal.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

struct RotaryArgs {
    const void *q, *k;
    void *qo, *ko;
    const float* table;
    const int64_t* positions;
    int64_t tokens, T, table_rows;
    int64_t qs[3], ks[3];    // strides of batch, token and head, in elements
    int64_t pos_b, pos_t;
    int Hq, H, D, R;         // H: query and key heads together
    int units, hslots, iters, tpb;
    float sign;
};

// V elements from p: one access of 16 bytes, or of 8 (four 16-bit values), or one
// value.
template <int DT, int V>
__device__ __forceinline__ void get(const void* p, int64_t i, float* f) {
    using E = Elem<DT>;
    const auto* q = reinterpret_cast<const typename E::S*>(p) + i;
    if constexpr (V == 1) {
        f[0] = E::to_f(q[0]);
    } else if constexpr (V == E::V) {
        E::unpack(*reinterpret_cast<const u32x4*>(q), f);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(q);
        float x[8];
        E::unpack(u32x4{w.x, w.y, 0, 0}, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = x[j];
    }
}
template <int DT, int V>
__device__ __forceinline__ void put(void* p, int64_t i, const float* f) {
    using E = Elem<DT>;
    auto* q = reinterpret_cast<typename E::S*>(p) + i;
    if constexpr (V == 1) {
        q[0] = E::from_f(f[0]);
    } else if constexpr (V == E::V) {
        *reinterpret_cast<u32x4*>(q) = E::pack(f);
    } else {
        const float x[8] = {f[0], f[1], f[2], f[3]};
        const u32x4 w = E::pack(x);
        *reinterpret_cast<uint2*>(q) = make_uint2(w.x, w.y);
    }
}

// A unit is two vectors of V elements of a head: at d and d + R/2 in the half
// layout's rotated part, neighbours elsewhere.  blockDim = units * hslots *
// tpb (whole waves): unit, head slot and token of the thread.
template <int DT, int V, bool INTER>
__global__ void rotary_kernel(RotaryArgs a) {
    const int u = threadIdx.x % a.units, rest = threadIdx.x / a.units;
    const int hs = rest % a.hslots, tl = rest / a.hslots;
    const int64_t token = (int64_t)blockIdx.x * a.tpb + tl;
    if (tl >= a.tpb || token >= a.tokens) return;
    const int64_t b = token / a.T, t = token - b * a.T;
    const int half = a.R >> 1, rot_units = INTER ? 0 : half / V;
    int d0, d1;
    bool r0, r1;
    if (!INTER && u < rot_units) {
        d0 = u * V; d1 = d0 + half; r0 = r1 = true;
    } else {
        d0 = (INTER ? 0 : a.R) + (u - rot_units) * 2 * V; d1 = d0 + V;
        r0 = INTER && d0 < a.R; r1 = INTER && d1 < a.R;
    }
    const int64_t pos = a.positions ? a.positions[b * a.pos_b + t * a.pos_t] : t;
    // a position outside the table gives NaN, never a read outside it
    const bool known = pos >= 0 && pos < a.table_rows;
    float c[V], s[V];   // interleaved: V/2 pairs of the first vector, then of the second
#pragma unroll
    for (int i = 0; i < V; ++i) { c[i] = 1.0f; s[i] = 0.0f; }
    const float* row = a.table + (known ? pos : 0) * a.R;
    if constexpr (!INTER) {
        if (r0) {
            if constexpr (V == 1) { c[0] = row[d0]; s[0] = row[half + d0]; }
            else {
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    Elem<AXS6_F32>::unpack(*reinterpret_cast<const u32x4*>(row + d0 + i), c + i);
                    Elem<AXS6_F32>::unpack(*reinterpret_cast<const u32x4*>(row + half + d0 + i), s + i);
                }
            }
        }
    } else if constexpr (V == 1) {
        if (r0) { c[0] = row[d0 >> 1]; s[0] = row[half + (d0 >> 1)]; }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int d = d0 + 2 * i;   // first value of pair i of the unit
            if (d < a.R) { c[i] = row[d >> 1]; s[i] = row[half + (d >> 1)]; }
        }
    }
    if ((r0 || r1) && !known) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!INTER || V == 1 || d0 + 2 * i < a.R) c[i] = __uint_as_float(0x7fc00000u);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= a.sign;
    for (int it = 0; it < a.iters; ++it) {
        const int h = (blockIdx.y * a.iters + it) * a.hslots + hs;
        if (h >= a.H) return;
        const bool isq = h < a.Hq;
        const int hh = isq ? h : h - a.Hq;
        const void* src = isq ? a.q : a.k;
        void* dst = isq ? a.qo : a.ko;
        const int64_t* st = isq ? a.qs : a.ks;
        const int64_t in = b * st[0] + t * st[1] + hh * st[2];
        const int64_t out = (token * (isq ? a.Hq : a.H - a.Hq) + hh) * a.D;
        float x[V], y[V];
        const bool two = d1 < a.D;
        get<DT, V>(src, in + d0, x);
        if (two) get<DT, V>(src, in + d1, y);
        if constexpr (!INTER || V == 1) {
            if (r0) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float p = x[i], q = y[i];
                    x[i] = p * c[i] - q * s[i];
                    y[i] = q * c[i] + p * s[i];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                if (r0) {
                    const float p = x[i], q = x[i + 1], cc = c[i / 2], ss = s[i / 2];
                    x[i] = p * cc - q * ss;
                    x[i + 1] = q * cc + p * ss;
                }
                if (r1) {
                    const float p = y[i], q = y[i + 1], cc = c[V / 2 + i / 2], ss = s[V / 2 + i / 2];
                    y[i] = p * cc - q * ss;
                    y[i + 1] = q * cc + p * ss;
                }
            }
        }
        put<DT, V>(dst, out + d0, x);
        if (two) put<DT, V>(dst, out + d1, y);
    }
}

constexpr int kRotaryThreads = 256;

template <int DT, bool INTER>
void launch(RotaryArgs a, int v, hipStream_t st) {
    a.units = INTER ? (a.D + 2 * v - 1) / (2 * v) : a.R / 2 / v + (a.D - a.R + 2 * v - 1) / (2 * v);
    const int most = kRotaryThreads / a.units;   // heads that a workgroup holds at once
    // up to 8 heads a thread where there are tokens enough to fill the chip without more threads
    int iters = (int)((a.tokens * a.H * a.units) / (256 * 1024));
    iters = iters < 1 ? 1 : iters > 8 ? 8 : iters;
    if (iters > a.H) iters = a.H;
    a.hslots = (a.H + iters - 1) / iters;
    if (a.hslots > most) a.hslots = most;
    a.iters = iters;
    a.tpb = kRotaryThreads / (a.units * a.hslots);
    if (a.tpb > a.tokens) a.tpb = (int)a.tokens;
    const int threads = (a.units * a.hslots * a.tpb + 63) / 64 * 64;
    const dim3 grid((unsigned)((a.tokens + a.tpb - 1) / a.tpb),
                    (unsigned)((a.H + a.hslots * a.iters - 1) / (a.hslots * a.iters)));
    if (v == Elem<DT>::V) rotary_kernel<DT, Elem<DT>::V, INTER><<<grid, threads, 0, st>>>(a);
    else if (v == 4) rotary_kernel<DT, 4, INTER><<<grid, threads, 0, st>>>(a);
    else rotary_kernel<DT, 1, INTER><<<grid, threads, 0, st>>>(a);
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int axs6_rotary(const void* q, const void* k, void* q_out, void* k_out, int32_t dtype, int64_t B, int64_t T,
                           int64_t Hq, int64_t Hkv, int64_t D, int64_t R, const int64_t* q_strides,
                           const int64_t* k_strides, const float* table, int64_t table_rows, const int64_t* positions,
                           int64_t pos_stride_b, int64_t pos_stride_t, int32_t interleaved, int32_t inverse,
                           void* stream) {
    const char* fn = "axs6_rotary";
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    if (B < 0 || T < 0 || Hq < 0 || Hkv < 0 || D < 0)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: negative dimension", fn);
    if (R < 0 || R % 2 || R > D)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: the rotated part of %lld values is not an even part of the head's %lld",
                    fn, (long long)R, (long long)D);
    if (D > 512) return fail(AXS6_ERR_UNSUPPORTED, "%s: heads of at most 512 values, got %lld", fn, (long long)D);
    if (Hq + Hkv > (1 << 20) || B > ((int64_t)1 << 31) || T > ((int64_t)1 << 31) || B * T > ((int64_t)1 << 31) - 1)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    if (!k) Hkv = 0;
    if (!q) Hq = 0;
    if (B * T == 0 || Hq + Hkv == 0 || D == 0) return AXS6_OK;
    if ((Hq && (!q_out || !q_strides)) || (Hkv && (!k_out || !k_strides)) || (R && !table) || table_rows < 0 ||
        (R && table_rows == 0))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null output, strides or table", fn);
    const int64_t es = dtype == AXS6_F32 ? 4 : 2;
    const void* ptrs[] = {q, q_out, k, k_out};
    for (const void* p : ptrs)
        if ((uintptr_t)p % es) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not element-aligned", fn);
    RotaryArgs a{};
    a.q = q; a.k = k; a.qo = q_out; a.ko = k_out; a.table = table; a.positions = positions;
    a.tokens = B * T; a.T = T; a.table_rows = table_rows;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = Hq ? q_strides[i] : 0;
        a.ks[i] = Hkv ? k_strides[i] : 0;
    }
    // The longest whole aligned vectors, none of which crosses a boundary of the
    // layout: 16 bytes; in 16 bits 8 (2 x 4096 tokens, 40 heads of 80, the first 40
    // values rotated in halves of 20: 20 us, by single values 44); a value.
    int v = (int)(16 / es);
    for (; v > 1; v = v == 8 ? 4 : 1) {
        bool whole = D % v == 0 && R % v == 0 && (interleaved || R / 2 % v == 0) && (uintptr_t)table % 16 == 0;
        for (const void* p : ptrs) whole = whole && (uintptr_t)p % (v * es) == 0;
        for (int i = 0; i < 3; ++i) whole = whole && a.qs[i] % v == 0 && a.ks[i] % v == 0;
        if (whole) break;
    }
    a.pos_b = pos_stride_b; a.pos_t = pos_stride_t;
    a.Hq = (int)Hq; a.H = (int)(Hq + Hkv); a.D = (int)D; a.R = (int)R;
    a.sign = inverse ? -1.0f : 1.0f;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case AXS6_F32: interleaved ? launch<AXS6_F32, true>(a, v, st) : launch<AXS6_F32, false>(a, v, st); break;
        case AXS6_BF16: interleaved ? launch<AXS6_BF16, true>(a, v, st) : launch<AXS6_BF16, false>(a, v, st); break;
        default: interleaved ? launch<AXS6_F16, true>(a, v, st) : launch<AXS6_F16, false>(a, v, st); break;
    }
    return check_launch(fn);
}
