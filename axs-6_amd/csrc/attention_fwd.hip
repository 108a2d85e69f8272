// Attention forward: o = softmax(scale q k^T + mask) v, heads of queries in
// groups that share a key head.
//
// With x_ij = scale q_i . k_j (and the mask), one pass over the keys keeps a
// row's running maximum m and sum l = sum_j exp(x_ij - m) and rescales the
// output when m grows; at the end o = sum_j exp(x_ij - m) v_j / l and
// lse = m + log l, the one number a row's probabilities are made from again in
// the backward.  A row that sees no key gives 0.
//
// Bound by the matrix cores (4 D operations a pair) and the exponentials
// beside them.  A wave holds 32 queries in registers; S^T = K q^T puts a
// query's scores in one lane and the lane 32 further on, so maximum and sum
// take one exchange, and the probabilities are the second product's operand
// in place.  A workgroup's four waves share the keys' tiles in LDS.
#include "attention.h"

namespace axs6 {
namespace {

constexpr int kFwdThreads = 256, kFwdQ = 128, kFwdK = 64;

template <int DT, int DC, bool MASK>
__global__ __launch_bounds__(kFwdThreads) void attn_fwd_kernel(AttnArgs a) {
    using T = Tile<DT, DC>;
    __shared__ __attribute__((aligned(16))) char kt[kFwdK * T::kPitch];
    __shared__ __attribute__((aligned(16))) char vt[kFwdK * T::kPitch];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int heads = a.B * a.Hq, bh = blockIdx.x % heads, b = bh / a.Hq, hq = bh % a.Hq, h = hq / a.G;
    const int q0 = ((int)(gridDim.x / heads) - 1 - (int)(blockIdx.x / heads)) * kFwdQ;   // a causal mask's longest rows first
    const int q = q0 + 32 * w + (lane & 31), qr = q < a.Tq ? q : a.Tq - 1;
    const int off = a.Tk - a.Tq;
    const int q_last = q0 + kFwdQ < a.Tq ? q0 + kFwdQ - 1 : a.Tq - 1;
    int keys = a.causal ? q_last + off + 1 : a.Tk;
    keys = keys < 0 ? 0 : keys > a.Tk ? a.Tk : keys;
    const int tiles = (keys + kFwdK - 1) / kFwdK;
    const int limit = a.causal ? (qr + off + 1 < a.Tk ? qr + off + 1 : a.Tk) : a.Tk;   // keys that the lane's row sees
    const int free_keys = a.causal ? q0 + off + 1 : a.Tk;   // below it every row of the workgroup sees every key

    const char* kb = reinterpret_cast<const char*>(a.k) + (b * a.ks[0] + h * a.ks[2]) * T::kBytes;
    const char* vb = reinterpret_cast<const char*>(a.v) + (b * a.vs[0] + h * a.vs[2]) * T::kBytes;
    const char* mrow = MASK ? mask_row(a, b, hq, qr) : nullptr;
    u32x4 qf[T::kSteps];
    load_rows<DT, DC>(qf, a.q, b * a.qs[0] + qr * a.qs[1] + hq * a.qs[2], a.D, lane);

    f32x16 o[DC / 32];
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.0f;
    const float c = a.scale * kLog2e;
    Stage<DT, DC, kFwdK, kFwdThreads> sk, sv;
    if (tiles) {
        sk.load(kb, a.ks[1], 0, a.Tk, a.D);
        sv.load(vb, a.vs[1], 0, a.Tk, a.D);
    }
    for (int t = 0; t < tiles; ++t) {
        __syncthreads();
        sk.store(kt);
        sv.store(vt);
        __syncthreads();
        const int k0 = t * kFwdK;
        if (t + 1 < tiles) {
            sk.load(kb, a.ks[1], k0 + kFwdK, a.Tk, a.D);
            sv.load(vb, a.vs[1], k0 + kFwdK, a.Tk, a.D);
        }
        f32x16 s[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            s[j] = zero16();
#pragma unroll
            for (int i = 0; i < T::kSteps; ++i) s[j] = mma<DT>(T::rows(kt, 32 * j, i, lane), qf[i], s[j]);
        }
        const bool whole = k0 + kFwdK <= free_keys && k0 + kFwdK <= a.Tk;
        float mx = m;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = k0 + 32 * j + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
                float x = s[j][i] * c;
                if constexpr (MASK) {
                    x = key < limit ? masked(a, mrow, key, x) : -INFINITY;
                } else if (!whole) {
                    x = key < limit ? x : -INFINITY;
                }
                s[j][i] = x;
                mx = fmaxf(mx, x);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        l *= alpha;
        u32x4 pf[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[j][i] = __builtin_amdgcn_exp2f(s[j][i] - ref);
                l += s[j][i];
            }
            fragments<DT>(s[j], pf[j]);
        }
#pragma unroll
        for (int d = 0; d < DC / 32; ++d) {
            o[d] *= alpha;
#pragma unroll
            for (int j = 0; j < 2; ++j) o[d] = T::cols(vt, 32 * j, d, s[j], pf[j], o[d], lane);
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (q >= a.Tq) return;
    const float rl = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t row = (((int64_t)b * a.Tq + q) * a.Hq + hq) * a.D;
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) store_cols<DT>(a.o, row, d, o[d], rl, a.D, lane);
    if (a.lse && lane < 32)
        a.lse[((int64_t)b * a.Hq + hq) * a.Tq + q] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

template <int DT, int DC>
void launch(const AttnArgs& a, hipStream_t st) {
    const unsigned grid = (unsigned)((a.Tq + kFwdQ - 1) / kFwdQ * a.B * a.Hq);
    if (a.mask) attn_fwd_kernel<DT, DC, true><<<grid, kFwdThreads, 0, st>>>(a);
    else attn_fwd_kernel<DT, DC, false><<<grid, kFwdThreads, 0, st>>>(a);
}

template <int DT>
void dispatch(const AttnArgs& a, hipStream_t st) {
    if (a.D <= 64) launch<DT, 64>(a, st);
    else if (a.D <= 96) launch<DT, 96>(a, st);
    else launch<DT, 128>(a, st);
}

// The arguments of both directions, checked.
int fill(const char* fn, AttnArgs& a, int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t H, int64_t D,
         const void* mask, int32_t mask_type, const int64_t* mask_strides, int32_t causal, float scale) {
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    if (B < 0 || Tq < 0 || Tk < 0 || Hq < 0 || H < 0)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: negative dimension", fn);
    if (H ? Hq % H != 0 : Hq != 0)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: %lld query heads for %lld key heads", fn, (long long)Hq, (long long)H);
    const int64_t v = dtype == AXS6_F32 ? 4 : 8;
    if (D <= 0 || D > AXS6_ATTENTION_MAX_HEAD || D % v)
        return fail(AXS6_ERR_UNSUPPORTED, "%s: heads of whole 16-byte vectors up to %d values, got %lld", fn,
                    AXS6_ATTENTION_MAX_HEAD, (long long)D);
    // a workgroup for every 128 queries or keys of a head, in one grid dimension
    if (Tq > ((int64_t)1 << 30) || Tk > ((int64_t)1 << 30) || B > ((int64_t)1 << 24) || Hq > ((int64_t)1 << 24) ||
        ((Tq > Tk ? Tq : Tk) / 128 + 1) * B * Hq > ((int64_t)1 << 30))
        return fail(AXS6_ERR_UNSUPPORTED, "%s: dimension too large", fn);
    if (!(scale > 0.0f) || !isfinite(scale))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: the scale must be positive and finite", fn);
    if (mask && ((mask_type != -1 && !valid_dtype(mask_type)) || !mask_strides))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: bad mask type or null strides", fn);
    a.mask = mask; a.mask_type = mask_type;
    for (int i = 0; i < 4; ++i) a.ms[i] = mask ? mask_strides[i] : 0;
    a.B = (int)B; a.Hq = (int)Hq; a.H = (int)H; a.G = H ? (int)(Hq / H) : 1; a.Tq = (int)Tq; a.Tk = (int)Tk;
    a.D = (int)D; a.causal = causal; a.scale = scale;
    return AXS6_OK;
}

// Pointer and strides of one operand: whole aligned 16-byte vectors.
int operand(const char* fn, const char* name, const void* p, const int64_t* strides, int dtype, int64_t* to) {
    if (!p || !strides) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null %s", fn, name);
    const int64_t v = dtype == AXS6_F32 ? 4 : 8;
    if ((uintptr_t)p % 16) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: %s not aligned to 16 bytes", fn, name);
    for (int i = 0; i < 3; ++i) {
        if (strides[i] % v) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: a stride of %s is not whole vectors", fn, name);
        to[i] = strides[i];
    }
    return AXS6_OK;
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int axs6_attention_forward(const void* q, const void* k, const void* v, int32_t dtype, int64_t B, int64_t Tq,
                                      int64_t Tk, int64_t Hq, int64_t H, int64_t D, const int64_t* q_strides,
                                      const int64_t* k_strides, const int64_t* v_strides, const void* mask,
                                      int32_t mask_type, const int64_t* mask_strides, int32_t causal, float scale,
                                      void* out, float* lse, void* stream) {
    const char* fn = "axs6_attention_forward";
    AttnArgs a{};
    int rc = fill(fn, a, dtype, B, Tq, Tk, Hq, H, D, mask, mask_type, mask_strides, causal, scale);
    if (rc) return rc;
    if (B * Tq * Hq == 0) return AXS6_OK;
    if ((rc = operand(fn, "q", q, q_strides, dtype, a.qs))) return rc;
    if (Tk && ((rc = operand(fn, "k", k, k_strides, dtype, a.ks)) || (rc = operand(fn, "v", v, v_strides, dtype, a.vs))))
        return rc;
    if (!out || (uintptr_t)out % 16) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: output null or not aligned", fn);
    a.q = q; a.k = k; a.v = v; a.o = out; a.lse = lse;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AXS6_F32) dispatch<AXS6_F32>(a, st);
    else if (dtype == AXS6_BF16) dispatch<AXS6_BF16>(a, st);
    else dispatch<AXS6_F16>(a, st);
    return check_launch(fn);
}

extern "C" int axs6_attention_backward(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                       const float* lse, int32_t dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
                                       int64_t H, int64_t D, const int64_t* dout_strides, const int64_t* q_strides,
                                       const int64_t* k_strides, const int64_t* v_strides, const void* mask,
                                       int32_t mask_type, const int64_t* mask_strides, int32_t causal, float scale,
                                       float* delta, void* dq, void* dk, void* dv, void* stream) {
    const char* fn = "axs6_attention_backward";
    AttnArgs a{};
    int rc = fill(fn, a, dtype, B, Tq, Tk, Hq, H, D, mask, mask_type, mask_strides, causal, scale);
    if (rc) return rc;
    if (B * Hq == 0 || (Tq == 0 && Tk == 0)) return AXS6_OK;
    const int64_t os[3] = {Tq * Hq * D, Hq * D, D};
    if (Tq && ((rc = operand(fn, "q", q, q_strides, dtype, a.qs)) ||
               (rc = operand(fn, "dout", dout, dout_strides, dtype, a.gs)) ||
               (rc = operand(fn, "out", out, os, dtype, a.os))))
        return rc;
    if (Tk && ((rc = operand(fn, "k", k, k_strides, dtype, a.ks)) || (rc = operand(fn, "v", v, v_strides, dtype, a.vs))))
        return rc;
    if ((Tq && (!lse || !delta || !dq)) || (Tk && (!dk || !dv)))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null lse, delta or gradient", fn);
    if ((uintptr_t)dq % 16 || (uintptr_t)dk % 16 || (uintptr_t)dv % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: gradients not aligned to 16 bytes", fn);
    a.q = q; a.k = k; a.v = v; a.out = out; a.dout = dout; a.lse = const_cast<float*>(lse); a.delta = delta;
    a.dq = dq; a.dk = dk; a.dv = dv;
    attention_backward(a, dtype, (hipStream_t)stream);
    return check_launch(fn);
}
