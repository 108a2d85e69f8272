// Attention backward: the gradients of queries, keys and values from the
// output's, with the probabilities made again from each row's lse.
//
//   p_ij = exp(x_ij - lse_i),  dv_j = sum_i p_ij do_i,
//   ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = sum_j p_ij do_i . v_j = do_i . o_i,
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i  (over the group's heads).
//
// Two launches, both without atomics, so that the sums have a fixed order.
// The first holds 32 queries a wave and walks over the keys (dq, and delta for
// the second); the second holds 32 keys a wave and walks over the queries of
// all heads of the group (dk, dv).  Scores and do . v are computed in both: 7
// products a pair instead of 5.
#include "attention.h"

namespace axs6 {
namespace {

constexpr int kBwdThreads = 256, kBwdHeld = 128, kBwdWalk = 32;

// dq of 128 queries; the loop is the forward's.
template <int DT, int DC, bool MASK>
__global__ __launch_bounds__(kBwdThreads) void attn_dq_kernel(AttnArgs a) {
    using T = Tile<DT, DC>;
    __shared__ __attribute__((aligned(16))) char kt[kBwdWalk * T::kPitch];
    __shared__ __attribute__((aligned(16))) char vt[kBwdWalk * T::kPitch];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int heads = a.B * a.Hq, bh = blockIdx.x % heads, b = bh / a.Hq, hq = bh % a.Hq, h = hq / a.G;
    const int q0 = ((int)(gridDim.x / heads) - 1 - (int)(blockIdx.x / heads)) * kBwdHeld;
    const int q = q0 + 32 * w + (lane & 31), qr = q < a.Tq ? q : a.Tq - 1;
    const int off = a.Tk - a.Tq;
    const int q_last = q0 + kBwdHeld < a.Tq ? q0 + kBwdHeld - 1 : a.Tq - 1;
    int keys = a.causal ? q_last + off + 1 : a.Tk;
    keys = keys < 0 ? 0 : keys > a.Tk ? a.Tk : keys;
    const int tiles = (keys + kBwdWalk - 1) / kBwdWalk;
    const int limit = a.causal ? (qr + off + 1 < a.Tk ? qr + off + 1 : a.Tk) : a.Tk;
    const int free_keys = a.causal ? q0 + off + 1 : a.Tk;

    const char* kb = reinterpret_cast<const char*>(a.k) + (b * a.ks[0] + h * a.ks[2]) * T::kBytes;
    const char* vb = reinterpret_cast<const char*>(a.v) + (b * a.vs[0] + h * a.vs[2]) * T::kBytes;
    const char* mrow = MASK ? mask_row(a, b, hq, qr) : nullptr;
    u32x4 qf[T::kSteps], gf[T::kSteps];
    load_rows<DT, DC>(qf, a.q, b * a.qs[0] + qr * a.qs[1] + hq * a.qs[2], a.D, lane);
    load_rows<DT, DC>(gf, a.dout, b * a.gs[0] + qr * a.gs[1] + hq * a.gs[2], a.D, lane);
    const int64_t row = ((int64_t)b * a.Hq + hq) * a.Tq + qr;
    float delta = 0.0f;
    {
        u32x4 of[T::kSteps];
        load_rows<DT, DC>(of, a.out, b * a.os[0] + qr * a.os[1] + hq * a.os[2], a.D, lane);
#pragma unroll
        for (int s = 0; s < T::kSteps; ++s) {
            float x[T::kVals], y[T::kVals];
            Elem<DT>::unpack(gf[s], x);
            Elem<DT>::unpack(of[s], y);
#pragma unroll
            for (int i = 0; i < T::kVals; ++i) delta += x[i] * y[i];
        }
        delta += __shfl_xor(delta, 32, 64);
        if (lane < 32 && q < a.Tq) a.delta[row] = delta;
    }
    const float lse = a.lse[row], c = a.scale * kLog2e;

    f32x16 dq[DC / 32];
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) dq[d] = zero16();
    Stage<DT, DC, kBwdWalk, kBwdThreads> sk, sv;
    if (tiles) {
        sk.load(kb, a.ks[1], 0, a.Tk, a.D);
        sv.load(vb, a.vs[1], 0, a.Tk, a.D);
    }
    for (int t = 0; t < tiles; ++t) {
        __syncthreads();
        sk.store(kt);
        sv.store(vt);
        __syncthreads();
        const int k0 = t * kBwdWalk;
        if (t + 1 < tiles) {
            sk.load(kb, a.ks[1], k0 + kBwdWalk, a.Tk, a.D);
            sv.load(vb, a.vs[1], k0 + kBwdWalk, a.Tk, a.D);
        }
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int i = 0; i < T::kSteps; ++i) s = mma<DT>(T::rows(kt, 0, i, lane), qf[i], s);
#pragma unroll
        for (int i = 0; i < T::kSteps; ++i) dp = mma<DT>(T::rows(vt, 0, i, lane), gf[i], dp);
        const bool whole = k0 + kBwdWalk <= free_keys && k0 + kBwdWalk <= a.Tk;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = k0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
            float x = s[i] * c;
            if constexpr (MASK) x = key < limit ? masked(a, mrow, key, x) : -INFINITY;
            else if (!whole) x = key < limit ? x : -INFINITY;
            s[i] = __builtin_amdgcn_exp2f(x - lse) * (dp[i] - delta);
        }
        u32x4 pf[2];
        fragments<DT>(s, pf);
#pragma unroll
        for (int d = 0; d < DC / 32; ++d) dq[d] = T::cols(kt, 0, d, s, pf, dq[d], lane);
    }
    if (q >= a.Tq) return;
    const int64_t out = (((int64_t)b * a.Tq + q) * a.Hq + hq) * a.D;
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) store_cols<DT>(a.dq, out, d, dq[d], a.scale, a.D, lane);
}

// dk and dv of 128 keys of one key head.
template <int DT, int DC, bool MASK>
__global__ __launch_bounds__(kBwdThreads) void attn_dkv_kernel(AttnArgs a) {
    using T = Tile<DT, DC>;
    __shared__ __attribute__((aligned(16))) char qt[kBwdWalk * T::kPitch];
    __shared__ __attribute__((aligned(16))) char gt[kBwdWalk * T::kPitch];
    __shared__ __attribute__((aligned(16))) float lt[kBwdWalk], dt[kBwdWalk];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int heads = a.B * a.H, bh = blockIdx.x % heads, b = bh / a.H, h = bh % a.H;
    const int k0 = blockIdx.x / heads * kBwdHeld;   // the first keys have the most queries under a causal mask
    const int key = k0 + 32 * w + (lane & 31), kr = key < a.Tk ? key : a.Tk - 1;
    const int off = a.Tk - a.Tq;
    int q_first = a.causal ? k0 - off : 0;   // the first query that sees one of the keys
    q_first = q_first < 0 ? 0 : q_first / kBwdWalk * kBwdWalk;
    const int per_head = q_first < a.Tq ? (a.Tq - q_first + kBwdWalk - 1) / kBwdWalk : 0;
    const int tiles = per_head * a.G;
    const int free_q = a.causal ? k0 + kBwdHeld - 1 - off : 0;   // from here on every query sees every key held

    u32x4 kf[T::kSteps], vf[T::kSteps];
    load_rows<DT, DC>(kf, a.k, b * a.ks[0] + kr * a.ks[1] + h * a.ks[2], a.D, lane);
    load_rows<DT, DC>(vf, a.v, b * a.vs[0] + kr * a.vs[1] + h * a.vs[2], a.D, lane);
    f32x16 dk[DC / 32], dv[DC / 32];
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
    const float c = a.scale * kLog2e;
    Stage<DT, DC, kBwdWalk, kBwdThreads> sq, sg;
    float sl = INFINITY, sd = 0.0f;
    auto load = [&](int t) {
        const int hq = h * a.G + t / per_head, i0 = q_first + t % per_head * kBwdWalk;
        sq.load(reinterpret_cast<const char*>(a.q) + (b * a.qs[0] + hq * a.qs[2]) * T::kBytes, a.qs[1], i0, a.Tq, a.D);
        sg.load(reinterpret_cast<const char*>(a.dout) + (b * a.gs[0] + hq * a.gs[2]) * T::kBytes, a.gs[1], i0, a.Tq, a.D);
        if (threadIdx.x < kBwdWalk) {
            const int i = i0 + threadIdx.x;
            const int64_t row = ((int64_t)b * a.Hq + hq) * a.Tq + i;
            sl = i < a.Tq ? a.lse[row] : INFINITY;   // rows past the end have no probabilities
            sd = i < a.Tq ? a.delta[row] : 0.0f;
        }
    };
    if (tiles) load(0);
    for (int t = 0; t < tiles; ++t) {
        __syncthreads();
        sq.store(qt);
        sg.store(gt);
        if (threadIdx.x < kBwdWalk) { lt[threadIdx.x] = sl; dt[threadIdx.x] = sd; }
        __syncthreads();
        const int hq = h * a.G + t / per_head, i0 = q_first + t % per_head * kBwdWalk;
        if (t + 1 < tiles) load(t + 1);
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int i = 0; i < T::kSteps; ++i) s = mma<DT>(T::rows(qt, 0, i, lane), kf[i], s);
#pragma unroll
        for (int i = 0; i < T::kSteps; ++i) dp = mma<DT>(T::rows(gt, 0, i, lane), vf[i], dp);
        const bool whole = i0 >= free_q;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 lse = *reinterpret_cast<const float4*>(lt + 8 * g + 4 * (lane >> 5));
            const float4 del = *reinterpret_cast<const float4*>(dt + 8 * g + 4 * (lane >> 5));
            const float ls[4] = {lse.x, lse.y, lse.z, lse.w}, ds[4] = {del.x, del.y, del.z, del.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * g + e, q = i0 + 8 * g + 4 * (lane >> 5) + e;
                float x = s[i] * c;
                if constexpr (MASK) {
                    const int qr = q < a.Tq ? q : a.Tq - 1;
                    x = !a.causal || kr <= q + off ? masked(a, mask_row(a, b, hq, qr), kr, x) : -INFINITY;
                } else if (!whole) {
                    x = kr <= q + off ? x : -INFINITY;
                }
                s[i] = __builtin_amdgcn_exp2f(x - ls[e]);
                dp[i] = s[i] * (dp[i] - ds[e]);
            }
        }
        u32x4 pf[2], df[2];
        fragments<DT>(s, pf);
        fragments<DT>(dp, df);
#pragma unroll
        for (int d = 0; d < DC / 32; ++d) {
            dv[d] = T::cols(gt, 0, d, s, pf, dv[d], lane);
            dk[d] = T::cols(qt, 0, d, dp, df, dk[d], lane);
        }
    }
    if (key >= a.Tk) return;
    const int64_t out = (((int64_t)b * a.Tk + key) * a.H + h) * a.D;
#pragma unroll
    for (int d = 0; d < DC / 32; ++d) {
        store_cols<DT>(a.dk, out, d, dk[d], a.scale, a.D, lane);
        store_cols<DT>(a.dv, out, d, dv[d], 1.0f, a.D, lane);
    }
}

template <int DT, int DC>
void launch(const AttnArgs& a, hipStream_t st) {
    if (a.Tq) {
        const unsigned grid = (unsigned)((a.Tq + kBwdHeld - 1) / kBwdHeld * a.B * a.Hq);
        if (a.mask) attn_dq_kernel<DT, DC, true><<<grid, kBwdThreads, 0, st>>>(a);
        else attn_dq_kernel<DT, DC, false><<<grid, kBwdThreads, 0, st>>>(a);
    }
    if (a.Tk) {
        const unsigned grid = (unsigned)((a.Tk + kBwdHeld - 1) / kBwdHeld * a.B * a.H);
        if (a.mask) attn_dkv_kernel<DT, DC, true><<<grid, kBwdThreads, 0, st>>>(a);
        else attn_dkv_kernel<DT, DC, false><<<grid, kBwdThreads, 0, st>>>(a);
    }
}

template <int DT>
void dispatch(const AttnArgs& a, hipStream_t st) {
    if (a.D <= 64) launch<DT, 64>(a, st);
    else if (a.D <= 96) launch<DT, 96>(a, st);
    else launch<DT, 128>(a, st);
}

}  // namespace

int attention_backward(const AttnArgs& a, int dtype, hipStream_t st) {
    if (dtype == AXS6_F32) dispatch<AXS6_F32>(a, st);
    else if (dtype == AXS6_BF16) dispatch<AXS6_BF16>(a, st);
    else dispatch<AXS6_F16>(a, st);
    return AXS6_OK;
}

}  // namespace axs6
