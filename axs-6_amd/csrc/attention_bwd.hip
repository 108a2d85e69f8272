// Attention backward: the gradients of queries, keys and values from the
// output's, with the probabilities made again from each row's maximum m and sum l.
//
//   p_ij = exp(x_ij - m_i - log l_i),  dv_j = sum_i p_ij do_i,
//   ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = sum_j p_ij do_i . v_j = do_i . o_i,
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i  (over the group's heads).
//
// Two launches, both without atomics, so that the sums have a fixed order.
// The first holds 32 queries a wave and walks over the keys (dq, and delta for
// the second); the second holds 32 keys a wave and walks over the queries of
// all heads of the group (dk, dv).  Scores and do . v are computed in both: 7
// products a pair instead of 5.  Tiles travel as in the forward.
// Under a causal mask the first keys are seen by far more queries than the
// last: their queries are split over workgroups, whose float32 sums a third
// launch adds (1 x 16384, 2 key heads for 16, bf16: 9072 -> 3824 us for both
// launches; 2 x 4096, 8 for 32: 1511 -> 1127, now 1020, of which dq 391: the 7
// products' 9.6e11 operations at 943 TFLOP/s, 83% of a bf16 product of 8192^3).
// A head of up to 64 values whose queries and keys are at most 128 is one
// workgroup's: the second launch then makes dq too, from ds by way of LDS, 5
// products instead of 7 and one launch instead of two.  64 x 128, 4 heads, causal:
// float32 61 -> 44 us, bf16 20 either way; 512 x 128: float32 431 -> 338, bf16 97 -> 101,
// float16 102 -> 98; 64 x 32 queries of 77 keys, 8 heads: 67 -> 37, bf16 16 -> 13.  (Larger heads' keys and scores
// leave no room for a second workgroup on the CU, or for the first.)  In float32 what
// is left is the wave's own chain: its 640 products of 64 cycles are 17 us of the 44.
#include "attention.h"

namespace axs6 {
namespace {

constexpr int kWaves = 4, kThr = 64 * kWaves, kHeld = 32 * kWaves;

// float16 has 2^-14 as its smallest normal value and 65504 as its largest: probabilities
// and score gradients go into their products times a power of two, which costs nothing
// inside the loops and is undone with the results' factors.
//  * dq: a query's score gradients times 2^3 / |do_i| (the power of two above it): ds is
//    normal down to p = 2^-17 beside values of 1, and in range for values of norm 4000.
//  * dk, dv: both times 2^e, e in 0 .. 15 and as large as leaves ds_ij, at most
//    p (|do_i| |v_j| + |delta_i|), below 2^15 for the keys held and all queries of the
//    group; the first launch leaves their largest |do| and |delta|.  e goes into the rows' y.
//    (A scale that follows the largest ds so far: 2 x 4096, 32 heads on 8, 1065 -> 1420 us.)
//  * Up to 128 keys (the form of one workgroup a head): as they are, p is large enough.
// 4096 keys, do of 1e-4: dq off by 5e-2 without, 7e-3, its own rounding, with.
// A larger ds still overflows, and its rows are made again.  The other types have
// float32's range and no scale.
__device__ __forceinline__ float row_scale(float norm2) {
    return norm2 > 0.0f && norm2 < INFINITY ? ldexpf(1.0f, 3 - ((__builtin_amdgcn_frexp_expf(norm2) + 1) >> 1)) : 1.0f;
}
__device__ __forceinline__ float finite_or_0(float x) { return fabsf(x) < INFINITY ? x : 0.0f; }
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
__device__ __forceinline__ int64_t bound_at(const AttnArgs& a, int b, int hq, int q) {
    return ((int64_t)b * a.Hq + hq) * ((a.Tq + 31) >> 5) + (q >> 5);
}
// |x|^2 of rows in fragments, the lane's row is l % 32
template <int DT, int N>
__device__ __forceinline__ float norm2(const u32x4 (&f)[N]) {
    constexpr int V = 16 / kElemBytes<DT>;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float x[V];
        Elem<DT>::unpack(f[i], x);
#pragma unroll
        for (int j = 0; j < V; ++j) s += x[j] * x[j];
    }
    return s + __shfl_xor(s, 32, 64);
}

// dq of a query from the keys k0 .. k1 - 1 that it sees, one by one.
template <int DT>
__device__ void dq_row(const AttnArgs& a, int b, int hq, int q, int k0, int k1, int split, float2 st, float delta,
                       int lane) {
    const int h = hq / a.G;
    const float c = a.scale * kLog2e;
    const Two qv = load_two<DT>(a.q, b * a.qs[0] + q * a.qs[1] + hq * a.qs[2], a.D, lane);
    const Two gv = load_two<DT>(a.dout, b * a.gs[0] + q * a.gs[1] + hq * a.gs[2], a.D, lane);
    Two r = {0.0f, 0.0f};
    for (int key = k0; key < k1 && !all_nan(r, a.D, lane); ++key) {
        const float f = pair_term(a, b, hq, q, key);
        if (f == -INFINITY) continue;
        const Two kv = load_two<DT>(a.k, b * a.ks[0] + key * a.ks[1] + h * a.ks[2], a.D, lane);
        const Two vv = load_two<DT>(a.v, b * a.vs[0] + key * a.vs[1] + h * a.vs[2], a.D, lane);
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(dot(qv, kv), c, f) - st.x - st.y);
        const float ds = p * (dot(gv, vv) - delta);
        r = {r.x + ds * kv.x, r.y + ds * kv.y};
    }
    r = {r.x * a.scale, r.y * a.scale};
    const int64_t out = (((int64_t)b * a.Tq + q) * a.Hq + hq) * a.D;
    if (a.splits > 1) store_two<AXS6_F32>(a.part + split * ((int64_t)a.B * a.Tq * a.Hq * a.D), out, r, a.D, lane);
    else store_two<DT>(a.dq, out, r, a.D, lane);
}

// dk and dv of a key from the queries of the group's tiles first .. tiles - 1
// that see it, one by one.
template <int DT, int kWalk>
__device__ void dkv_row(const AttnArgs& a, int b, int h, int key, int first, int tiles, int q_first, int per_head,
                        int split, int lane) {
    const float c = a.scale * kLog2e;
    const Two kv = load_two<DT>(a.k, b * a.ks[0] + key * a.ks[1] + h * a.ks[2], a.D, lane);
    const Two vv = load_two<DT>(a.v, b * a.vs[0] + key * a.vs[1] + h * a.vs[2], a.D, lane);
    Two rk = {0.0f, 0.0f}, rv = {0.0f, 0.0f};
    for (int t = first; t < tiles && !(all_nan(rk, a.D, lane) && all_nan(rv, a.D, lane)); ++t) {
        const int hq = h * a.G + t / per_head, i0 = q_first + t % per_head * kWalk;
        for (int q = i0; q < i0 + kWalk && q < a.Tq; ++q) {
            const float f = pair_term(a, b, hq, q, key);
            if (f == -INFINITY) continue;
            const int64_t row = ((int64_t)b * a.Hq + hq) * a.Tq + q;
            const Two qv = load_two<DT>(a.q, b * a.qs[0] + q * a.qs[1] + hq * a.qs[2], a.D, lane);
            const Two gv = load_two<DT>(a.dout, b * a.gs[0] + q * a.gs[1] + hq * a.gs[2], a.D, lane);
            const float2 st = a.stats[row];
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(dot(qv, kv), c, f) - st.x - st.y);
            const float ds = p * (dot(gv, vv) - a.delta[row]);
            rk = {rk.x + ds * qv.x, rk.y + ds * qv.y};
            rv = {rv.x + p * gv.x, rv.y + p * gv.y};
        }
    }
    rk = {rk.x * a.scale, rk.y * a.scale};
    const int64_t out = (((int64_t)b * a.Tk + key) * a.H + h) * a.D;
    if (a.splits_kv > 1) {
        const int64_t all = (int64_t)a.B * a.Tk * a.H * a.D;
        store_two<AXS6_F32>(a.part_kv + split * all, out, rk, a.D, lane);
        store_two<AXS6_F32>(a.part_kv + (a.splits_kv + split) * all, out, rv, a.D, lane);
    } else {
        store_two<DT>(a.dk, out, rk, a.D, lane);
        store_two<DT>(a.dv, out, rv, a.D, lane);
    }
}

template <int DT, int DC> struct DqShape {
    static constexpr int kKeys = DT == AXS6_F32 ? 32 : 64;
    static constexpr int kOccupancy = DT == AXS6_F32 ? 1 : 2;
};

// dq of 128 queries; the loop is the forward's.
template <int DT, int DC, int MASK>
__global__ __launch_bounds__(kThr, (DqShape<DT, DC>::kOccupancy)) void attn_dq_kernel(AttnArgs a) {
    using T = Tile<DT, DC>;
    constexpr int KEYS = DqShape<DT, DC>::kKeys, NK = KEYS / 32;
    __shared__ __attribute__((aligned(1024))) char kt[2][KEYS * T::kPitch];
    __shared__ __attribute__((aligned(1024))) char vt[2][KEYS * T::kPitch];
    __shared__ __attribute__((aligned(16))) float term[2][by_key(MASK) ? KEYS : 1];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q_tiles = (a.Tq + kHeld - 1) / kHeld;
    int bh, piece;
    work_item(blockIdx.x, a.B * a.Hq, q_tiles * a.splits, a.causal, bh, piece);
    const int b = bh / a.Hq, hq = bh % a.Hq, h = hq / a.G, split = piece % a.splits;
    const int q0 = (q_tiles - 1 - piece / a.splits) * kHeld;
    const int off = a.Tk - a.Tq;
    const int q_last = q0 + kHeld < a.Tq ? q0 + kHeld - 1 : a.Tq - 1;
    int keys = a.causal ? q_last + off + 1 : a.Tk;
    keys = keys < 0 ? 0 : keys > a.Tk ? a.Tk : keys;
    int first = 0, tiles = (keys + KEYS - 1) / KEYS;
    if (a.splits > 1) {
        const int per = (tiles + a.splits - 1) / a.splits;
        first = split * per < tiles ? split * per : tiles;
        tiles = first + per < tiles ? first + per : tiles;
    }
    const int free_keys = a.causal ? q0 + off + 1 : a.Tk;
    const int free_tiles = free_keys <= 0 ? 0 : (free_keys < a.Tk ? free_keys : a.Tk) / KEYS;

    const char* kb = reinterpret_cast<const char*>(a.k) + (b * a.ks[0] + h * a.ks[2]) * T::kBytes;
    const char* vb = reinterpret_cast<const char*>(a.v) + (b * a.vs[0] + h * a.vs[2]) * T::kBytes;
    Direct<DT, DC, KEYS, kWaves> dk, dv;
    dk.init(a.ks[1], a.D, lane, w);
    dv.init(a.vs[1], a.D, lane, w);
    auto key_term = [&](int t) {
        const int key = t * KEYS + threadIdx.x;
        return threadIdx.x < KEYS && key < a.Tk ? mask_term(a, mask_row(a, b, hq, 0), key) : -INFINITY;
    };
    if (first < tiles) {
        dk.load(kt[first & 1], kb, first * KEYS, a.Tk, a.D, w);
        dv.load(vt[first & 1], vb, first * KEYS, a.Tk, a.D, w);
        if constexpr (by_key(MASK)) {
            const float f = key_term(first);
            if (threadIdx.x < KEYS) term[first & 1][threadIdx.x] = f;
        }
    }
    const int q = q0 + 32 * w + (lane & 31), qr = q < a.Tq ? q : a.Tq - 1;
    const int limit = a.causal && qr + off + 1 < a.Tk ? qr + off + 1 : a.Tk;
    const char* mrow = MASK == kFullMask ? mask_row(a, b, hq, qr) : nullptr;
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
        if (lane < 32 && q < a.Tq && split == 0) a.delta[row] = delta;
    }
    const float2 st = a.stats[row];
    const float lse = adds(MASK) ? st.x : st.x + st.y, c = a.scale * kLog2e;
    const bool apart = adds(MASK) && __any(st.y != 0.0f);

    f32x16 dq[T::kResults];
#pragma unroll
    for (int d = 0; d < T::kResults; ++d) dq[d] = zero16();
    float rs = 1.0f;   // the scale of the row's score gradients
    if constexpr (DT == AXS6_F16) {
        const float g2 = norm2<DT>(gf);
        rs = row_scale(g2);
        const bool here = lane < 32 && q < a.Tq;
        const float g = sqrtf(wave_max(here ? finite_or_0(g2) : 0.0f)), d = wave_max(here ? fabsf(finite_or_0(delta)) : 0.0f);
        if (lane == 0 && q < a.Tq && split == 0) a.bounds[bound_at(a, b, hq, q)] = make_float2(g, d);
    }
    const float delta_s = delta * rs;
    const bool rows_here = q0 + 32 * w < a.Tq;
    const int w_last = q0 + 32 * w + 31 < a.Tq ? q0 + 32 * w + 31 : a.Tq - 1;   // the wave's last row and its keys
    const int w_keys = a.causal && w_last + off + 1 < a.Tk ? w_last + off + 1 : a.Tk;
    for (int t = first; t < tiles; ++t) {
        tile_barrier();
        float next_term = 0.0f;
        if (t + 1 < tiles) {
            dk.load(kt[(t + 1) & 1], kb, (t + 1) * KEYS, a.Tk, a.D, w);
            dv.load(vt[(t + 1) & 1], vb, (t + 1) * KEYS, a.Tk, a.D, w);
            if constexpr (by_key(MASK)) next_term = key_term(t + 1);
        }
        const char *ks = kt[t & 1], *vs = vt[t & 1];
        const int k0 = t * KEYS;
        bool any = rows_here;
        bool plain = MASK == kNoMask;
        if constexpr (by_key(MASK)) {
            const float f = term[t & 1][lane & (KEYS - 1)];
            any = any && __any(!(f == -INFINITY));
            plain = __all(f == 0.0f);
        }
        const float cs = plain ? c : 1.0f;
        if (any) {
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                if (k0 + 32 * j >= w_keys) break;   // none of the wave's rows sees them
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int i = 0; i < T::kSteps; ++i) s = mma<DT>(T::rows(ks, 32 * j, i, lane), qf[i], s);
#pragma unroll
                for (int i = 0; i < T::kSteps; ++i) dp = mma<DT>(T::rows(vs, 32 * j, i, lane), gf[i], dp);
                apply_mask<MASK>(a, s, c, k0 + 32 * j, &term[t & 1][by_key(MASK) ? 32 * j : 0], mrow, plain,
                                 t >= free_tiles, limit, lane);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = __builtin_fmaf(s[i], cs, -lse);
                }
                if (apart)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] -= st.y;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(s[i]) * (DT == AXS6_F16 ? __builtin_fmaf(dp[i], rs, -delta_s) : dp[i] - delta);
                }
                u32x4 pf[2];
                fragments<DT>(s, pf);
                T::accumulate(ks, 32 * j, s, pf, dq, lane);
            }
        }
        if constexpr (by_key(MASK))
            if (threadIdx.x < KEYS) term[(t + 1) & 1][threadIdx.x] = next_term;
    }
    const bool bad = not_finite(dq);
    const int64_t out = (((int64_t)b * a.Tq + qr) * a.Hq + hq) * a.D;
    if (q < a.Tq) {
        float* part = a.part + split * ((int64_t)a.B * a.Tq * a.Hq * a.D);
        if (a.splits > 1) T::template store<AXS6_F32>(part, out, dq, a.scale / rs, a.D, lane);
        else T::template store<DT>(a.dq, out, dq, a.scale / rs, a.D, lane);
    }
    for (uint64_t rows = __ballot(bad && lane < 32 && q < a.Tq); rows; rows &= rows - 1) {
        const int r = __builtin_ctzll(rows);
        dq_row<DT>(a, b, hq, q0 + 32 * w + r, first * KEYS, tiles * KEYS < a.Tk ? tiles * KEYS : a.Tk, split,
                   make_float2(__shfl(st.x, r, 64), __shfl(st.y, r, 64)), __shfl(delta, r, 64), lane);
    }
}

template <int DT, int DC, int MASK, bool WHOLE> struct DkvShape {
    // the values held stay in LDS where their fragments would leave a wave more
    // than half of a SIMD's registers
    static constexpr bool kVInLds = DC > 96;
    // three waves a SIMD where 168 registers are enough (8 x 777, 12 heads of 64, a mask by
    // key: 127 -> 103 us for both launches)
    static constexpr int kOccupancy = DT == AXS6_F32 ? 1 : DC <= 64 && MASK != kFullMask && !WHOLE ? 3 : 2;
    // Queries of a tile that the held keys walk over: 64 for half the barriers, where
    // they and two waves fit (8 x 777, 12 heads of 80: 156 -> 148 us for both launches; 8 x 2048, 16
    // heads of 96: 843 -> 826; heads of 64, with two waves then for three, 95 -> 112)
    static constexpr int kWalk = DT != AXS6_F32 && DC > 64 && DC <= 96 && MASK != kFullMask ? 64 : 32;
};

// ds of a head's 128 queries and the 128 keys held, in the type, a query's keys
// one after another: the waves that made it hold keys, those that take it hold queries.
template <int DT>
struct Scores {
    using S = typename Elem<DT>::S;
    static constexpr int kPitch = kHeld + 16 / (int)sizeof(S);   // 16 bytes more: rows start at all banks
    // the 32 queries from q0 and the lane's key; df: ds in fragments (16-bit types)
    __device__ static void put(S* p, int q0, int key, const f32x16& ds, const u32x4 (&df)[2], int lane) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            S* x = p + (q0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)) * kPitch + key;
            if constexpr (DT == AXS6_F32) *x = ds[i];
            else *reinterpret_cast<uint16_t*>(x) = (uint16_t)(df[i >> 3][(i & 7) >> 1] >> (16 * (i & 1)));
        }
    }
    // the lane's query and the 32 keys from k0, as a result whose rows are the keys
    __device__ static void get(const S* p, int q, int k0, f32x16& ds, u32x4 (&df)[2], int lane) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const S* x = p + q * kPitch + k0 + 8 * g + 4 * (lane >> 5);
            if constexpr (DT == AXS6_F32) {
                const float4 v = *reinterpret_cast<const float4*>(x);
                ds[4 * g] = v.x; ds[4 * g + 1] = v.y; ds[4 * g + 2] = v.z; ds[4 * g + 3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(x);
                df[g >> 1][2 * (g & 1)] = v.x;
                df[g >> 1][2 * (g & 1) + 1] = v.y;
            }
        }
    }
};

// dk and dv of 128 keys of one key head.  WHOLE: there are no more keys and no more
// than 128 queries, and dq is made here too.
template <int DT, int DC, int MASK, bool WHOLE>
__global__ __launch_bounds__(kThr, (DkvShape<DT, DC, MASK, WHOLE>::kOccupancy)) void attn_dkv_kernel(AttnArgs a) {
    using T = Tile<DT, DC>;
    using S = Scores<DT>;
    constexpr bool VL = DkvShape<DT, DC, MASK, WHOLE>::kVInLds;
    constexpr int kWalk = DkvShape<DT, DC, MASK, WHOLE>::kWalk;
    __shared__ __attribute__((aligned(1024))) char kt[WHOLE ? kHeld * T::kPitch : 16];
    __shared__ __attribute__((aligned(16))) typename S::S scores[WHOLE ? kHeld * S::kPitch : 4];
    __shared__ __attribute__((aligned(1024))) char qt[2][kWalk * T::kPitch];
    __shared__ __attribute__((aligned(1024))) char gt[2][kWalk * T::kPitch];
    __shared__ __attribute__((aligned(1024))) char vt[VL ? kHeld * T::kPitch : 16];
    __shared__ __attribute__((aligned(16))) float lt[2][kWalk], dt[2][kWalk];
    // the rows' second numbers, and whether one of them is not 0
    __shared__ __attribute__((aligned(16))) float rt[2][adds(MASK) ? kWalk : 4];
    __shared__ int rest[2];
    constexpr bool kScaled = DT == AXS6_F16 && !WHOLE;
    __shared__ float4 largest[kScaled ? kWaves : 1];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int k_tiles = (a.Tk + kHeld - 1) / kHeld;
    int bh, piece;
    work_item(blockIdx.x, a.B * a.H, k_tiles * a.splits_kv, true, bh, piece);
    const int b = bh / a.H, h = bh % a.H, split = piece % a.splits_kv;
    const int k0 = piece / a.splits_kv * kHeld;   // the first keys have the most queries under a causal mask
    const int key = k0 + 32 * w + (lane & 31), kr = key < a.Tk ? key : a.Tk - 1;
    const int off = a.Tk - a.Tq;
    int q_first = a.causal ? k0 - off : 0;   // the first query that sees one of the keys
    q_first = q_first < 0 ? 0 : q_first / kWalk * kWalk;
    const int per_head = q_first < a.Tq ? (a.Tq - q_first + kWalk - 1) / kWalk : 0;
    int first = 0, tiles = per_head * a.G;   // the group's heads one after another
    if (a.splits_kv > 1) {
        const int per = (tiles + a.splits_kv - 1) / a.splits_kv;
        first = split * per < tiles ? split * per : tiles;
        tiles = first + per < tiles ? first + per : tiles;
    }
    const int free_q = a.causal ? k0 + kHeld - 1 - off : 0;   // from here on every query sees every key held

    Direct<DT, DC, kWalk, kWaves> lq, lg;
    lq.init(a.qs[1], a.D, lane, w);
    lg.init(a.gs[1], a.D, lane, w);
    const char* vb = reinterpret_cast<const char*>(a.v) + (b * a.vs[0] + h * a.vs[2]) * T::kBytes;
    if constexpr (VL) {
        Direct<DT, DC, kHeld, kWaves> lv;
        lv.init(a.vs[1], a.D, lane, w);
        lv.load(vt, vb, k0, a.Tk, a.D, w);
    }
    if constexpr (WHOLE) {
        Direct<DT, DC, kHeld, kWaves> lk;
        lk.init(a.ks[1], a.D, lane, w);
        lk.load(kt, reinterpret_cast<const char*>(a.k) + (b * a.ks[0] + h * a.ks[2]) * T::kBytes, 0, a.Tk, a.D, w);
    }
    // head and first query of the tile on its way
    int hq = h * a.G + (per_head ? first / per_head : 0), i0 = q_first + (per_head ? first % per_head : 0) * kWalk;
    float sl = 0.0f, sr = 0.0f, sd = 0.0f;
    float e = 0.0f;   // probabilities and score gradients are 2^e of themselves
    // WHOLE: out and dout of the tile's rows, eight threads a row, for its delta
    constexpr int N = DC / 8 / T::kVals;
    u32x4 xo[N], xg[N];
    int64_t row_on_way = -1;
    auto load = [&](char* qn, char* gn) {
        lq.load(qn, reinterpret_cast<const char*>(a.q) + (b * a.qs[0] + hq * a.qs[2]) * T::kBytes, i0, a.Tq, a.D, w);
        lg.load(gn, reinterpret_cast<const char*>(a.dout) + (b * a.gs[0] + hq * a.gs[2]) * T::kBytes, i0, a.Tq, a.D, w);
        if (threadIdx.x < kWalk) {
            const int i = i0 + threadIdx.x;
            const int64_t row = ((int64_t)b * a.Hq + hq) * a.Tq + i;
            const float2 st = i < a.Tq ? a.stats[row] : make_float2(INFINITY, 0.0f);   // rows past the end have no probabilities
            sl = adds(MASK) ? st.x : st.x + st.y;
            sr = st.y;
            if constexpr (!WHOLE) sd = i < a.Tq ? a.delta[row] : 0.0f;
        }
        if constexpr (WHOLE) {
            const int i = i0 + (threadIdx.x >> 3), d = (threadIdx.x & 7) * (DC / 8);
            row_on_way = i < a.Tq ? ((int64_t)b * a.Hq + hq) * a.Tq + i : -1;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                xo[e] = xg[e] = u32x4{0, 0, 0, 0};
                if (i < a.Tq && d + e * T::kVals < a.D) {
                    xo[e] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(a.out) +
                                                            (b * a.os[0] + i * a.os[1] + hq * a.os[2] + d + e * T::kVals) * T::kBytes);
                    xg[e] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(a.dout) +
                                                            (b * a.gs[0] + i * a.gs[1] + hq * a.gs[2] + d + e * T::kVals) * T::kBytes);
                }
            }
        }
    };
    auto store = [&](int buf) {
        if constexpr (kScaled) {
            // see row_stats: a large y has no place for e
            if (adds(MASK) && fabsf(sl) >= 128.0f && sl != INFINITY) sr -= e;
            else sl -= e;
        }
        if (threadIdx.x < kWalk) {
            lt[buf][threadIdx.x] = sl;
            if constexpr (adds(MASK)) {
                rt[buf][threadIdx.x] = sr;
                const bool some = __any(sr != 0.0f);
                if (threadIdx.x == 0) rest[buf] = some;
            }
            if constexpr (!WHOLE) dt[buf][threadIdx.x] = sd;
        }
        if constexpr (WHOLE) {
            float delta = 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float x[T::kVals], y[T::kVals];
                Elem<DT>::unpack(xo[e], x);
                Elem<DT>::unpack(xg[e], y);
#pragma unroll
                for (int i = 0; i < T::kVals; ++i) delta += x[i] * y[i];
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) delta += __shfl_xor(delta, o, 64);
            if ((threadIdx.x & 7) == 0) {
                dt[buf][threadIdx.x >> 3] = delta;
                if (row_on_way >= 0) a.delta[row_on_way] = delta;   // for rows made again
            }
        }
    };
    if (first < tiles) {
        if constexpr (kScaled) {
            // the largest |v| held, |do| and |delta| of the group's queries: on their way before the tiles
            const int n = (a.Tq + 31) >> 5, from = q_first >> 5, all = (n - from) * a.G;
            auto bound = [&](int i) {
                return i < all ? a.bounds[bound_at(a, b, h * a.G + i / (n - from), (from + i % (n - from)) * 32)]
                               : make_float2(0.0f, 0.0f);
            };
            u32x4 rows[T::kSteps];
            load_rows<DT, DC>(rows, a.v, b * a.vs[0] + kr * a.vs[1] + h * a.vs[2], a.D, lane);
            const float2 x = bound(threadIdx.x);
            load(qt[first & 1], gt[first & 1]);
            float3 m = make_float3(finite_or_0(norm2<DT>(rows)), x.x, x.y);
            for (int i = threadIdx.x + kThr; i < all; i += kThr) {
                const float2 y = bound(i);
                m.y = fmaxf(m.y, y.x);
                m.z = fmaxf(m.z, y.y);
            }
            m = make_float3(wave_max(m.x), wave_max(m.y), wave_max(m.z));
            if (lane == 0) largest[w] = make_float4(m.x, m.y, m.z, 0.0f);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                const float4 x = largest[i];
                m = make_float3(fmaxf(m.x, x.x), fmaxf(m.y, x.y), fmaxf(m.z, x.z));
            }
            e = (float)(15 - __builtin_amdgcn_frexp_expf(m.y * sqrtf(m.x) + m.z));
            e = fminf(fmaxf(e, 0.0f), 15.0f);
        } else {
            load(qt[first & 1], gt[first & 1]);
        }
        store(first & 1);
    }
    if constexpr (WHOLE)   // lanes past the last key hold a copy of it, which dq must not add again
        if (key >= a.Tk)
            for (int i = lane >> 5; i < kHeld; i += 2) scores[i * S::kPitch + key - k0] = typename S::S(0);
    u32x4 kf[T::kSteps], vf[VL ? 1 : T::kSteps];
    load_rows<DT, DC>(kf, a.k, b * a.ks[0] + kr * a.ks[1] + h * a.ks[2], a.D, lane);
    if constexpr (!VL) load_rows<DT, DC>(vf, a.v, b * a.vs[0] + kr * a.vs[1] + h * a.vs[2], a.D, lane);
    f32x16 dk[T::kResults], dv[T::kResults];
#pragma unroll
    for (int d = 0; d < T::kResults; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
    const float c = a.scale * kLog2e;
    float term = 0.0f;   // the mask's of the lane's key
    // The tile's buffers and the next one's are told apart by the parameters: the
    // compiler would else wait for the next tile before it reads this one.
    auto step = [&](int t, const char* __restrict__ qs, const char* __restrict__ gs, char* __restrict__ qn,
                    char* __restrict__ gn) __attribute__((always_inline)) {
        const int hq_now = hq, i_now = i0;
        if constexpr (by_key(MASK))
            if (t == first || i_now == q_first) term = mask_term(a, mask_row(a, b, hq_now, 0), kr);
        i0 += kWalk;
        if (i0 >= a.Tq) { i0 = q_first; ++hq; }
        if (t + 1 < tiles) load(qn, gn);
#pragma unroll
        for (int j = 0; j < kWalk / 32; ++j) {
            const int i_sub = i_now + 32 * j;
            if (j && i_sub >= a.Tq) break;
            // none of the 32 queries sees the wave's keys: they are before them, or the mask hides them
            bool any = !a.causal || i_sub + 31 + off >= k0 + 32 * w;
            if constexpr (by_key(MASK)) any = any && __any(!(term == -INFINITY));
            if (any) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int i = 0; i < T::kSteps; ++i) s = mma<DT>(T::rows(qs, 32 * j, i, lane), kf[i], s);
#pragma unroll
                for (int i = 0; i < T::kSteps; ++i) {
                    u32x4 v;
                    if constexpr (VL) v = T::rows(vt, 32 * w, i, lane);
                    else v = vf[i];
                    dp = mma<DT>(T::rows(gs, 32 * j, i, lane), v, dp);
                }
                const bool edge = i_sub < free_q;
                const int sub = 32 * j + 4 * (lane >> 5);
                // the rows' second numbers: for a full mask where one is not 0 (always: 8 x 1024 x 1024
                // scores of 128 values 330 -> 403 us), by key always (where one is not 0, which
                // takes registers of the whole loop: 8 x 777, 12 heads of 64 109 -> 120 us)
                const bool apart = MASK == kFullMask && __builtin_amdgcn_readfirstlane(rest[t & 1]);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 lse = *reinterpret_cast<const float4*>(&lt[t & 1][sub + 8 * g]);
                    const float4 del = *reinterpret_cast<const float4*>(&dt[t & 1][sub + 8 * g]);
                    const float ls[4] = {lse.x, lse.y, lse.z, lse.w}, ds[4] = {del.x, del.y, del.z, del.w};
                    float4 second = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if constexpr (MASK == kKeyAdd) second = *reinterpret_cast<const float4*>(&rt[t & 1][sub + 8 * g]);
                    const float rs[4] = {second.x, second.y, second.z, second.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * g + e, q = i_sub + 8 * g + 4 * (lane >> 5) + e;
                        float f = term;   // by key: the lane's
                        if constexpr (MASK == kFullMask)
                            f = mask_term(a, mask_row(a, b, hq_now, q < a.Tq ? q : a.Tq - 1), kr);
                        float x = __builtin_fmaf(s[i], c, adds(MASK) ? f : MASK == kNoMask ? -ls[e] : f - ls[e]);
                        if constexpr (adds(MASK)) x -= ls[e];
                        if constexpr (MASK == kKeyAdd) x -= rs[e];
                        if (apart) x -= rt[t & 1][sub + 8 * g + e];
                        if (edge) x = kr <= q + off ? x : -INFINITY;
                        s[i] = __builtin_amdgcn_exp2f(x);
                        dp[i] = s[i] * (dp[i] - ds[e]);
                    }
                }
                u32x4 pf[2], df[2];
                fragments<DT>(s, pf);
                fragments<DT>(dp, df);
                T::accumulate(gs, 32 * j, s, pf, dv, lane);
                T::accumulate(qs, 32 * j, dp, df, dk, lane);
                if constexpr (WHOLE)
                    if (key < a.Tk) S::put(scores, i_sub, key, dp, df, lane);
            } else if constexpr (WHOLE) {
                const u32x4 none[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                S::put(scores, i_sub, key, zero16(), none, lane);
            }
        }
        if (t + 1 < tiles) store((t + 1) & 1);
    };
    // WHOLE: dq of a head when its last tile is done; a wave takes 32 queries
    auto queries = [&](int head) {
        __syncthreads();
        const int q0 = 32 * w, q = q0 + (lane & 31);
        const int q_last = q0 + 31 < a.Tq ? q0 + 31 : a.Tq - 1;
        if (q0 >= a.Tq) return;
        f32x16 dq[T::kResults];
#pragma unroll
        for (int d = 0; d < T::kResults; ++d) dq[d] = zero16();
        const int keys = a.causal && q_last + off + 1 < a.Tk ? q_last + off + 1 : a.Tk;
        if (q0 >= q_first)   // those before see no key
            for (int j = 0; j < keys; j += 32) {
                f32x16 ds;
                u32x4 df[2];
                S::get(scores, q, j, ds, df, lane);
                T::accumulate(kt, j, ds, df, dq, lane);
            }
        const bool bad = not_finite(dq);
        if (q < a.Tq)
            T::template store<DT>(a.dq, (((int64_t)b * a.Tq + q) * a.Hq + head) * a.D, dq, a.scale, a.D, lane);
        for (uint64_t rows = __ballot(bad && lane < 32 && q < a.Tq); rows; rows &= rows - 1) {
            const int r = q0 + __builtin_ctzll(rows);
            const int64_t row = ((int64_t)b * a.Hq + head) * a.Tq + r;
            dq_row<DT>(a, b, head, r, 0, a.Tk, 0, a.stats[row], a.delta[row], lane);
        }
    };
    for (int t = first; t < tiles; ++t) {
        tile_barrier();
        const int head = hq;
        step(t, qt[t & 1], gt[t & 1], qt[(t + 1) & 1], gt[(t + 1) & 1]);
        if constexpr (WHOLE)
            if (hq != head) queries(head);
    }
    const bool bad = not_finite(dk) || not_finite(dv);
    const float fv = kScaled ? ldexpf(1.0f, -(int)e) : 1.0f, fk = a.scale * fv;
    if (key < a.Tk) {
        const int64_t out = (((int64_t)b * a.Tk + key) * a.H + h) * a.D, all = (int64_t)a.B * a.Tk * a.H * a.D;
        if (a.splits_kv > 1) {
            T::template store<AXS6_F32>(a.part_kv + split * all, out, dk, fk, a.D, lane);
            T::template store<AXS6_F32>(a.part_kv + (a.splits_kv + split) * all, out, dv, fv, a.D, lane);
        } else {
            T::template store<DT>(a.dk, out, dk, fk, a.D, lane);
            T::template store<DT>(a.dv, out, dv, fv, a.D, lane);
        }
    }
    for (uint64_t rows = __ballot(bad && lane < 32 && key < a.Tk); rows; rows &= rows - 1)
        dkv_row<DT, kWalk>(a, b, h, k0 + 32 * w + __builtin_ctzll(rows), first, tiles, q_first, per_head, split, lane);
}

// Sums of the splits in order, four values a thread; of two results, one after
// the other in part, in one launch.
template <int DT>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* part, int splits, int64_t n, void* out0, void* out1) {
    using E = Elem<DT>;
    void* out = blockIdx.y ? out1 : out0;
    part += blockIdx.y * splits * n;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float4 x = *reinterpret_cast<const float4*>(part + i);
    for (int s = 1; s < splits; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(part + s * n + i);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    auto* p = reinterpret_cast<typename E::S*>(out) + i;
    if constexpr (DT == AXS6_F32) *reinterpret_cast<float4*>(p) = x;
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<DT>(x.x, x.y), pack2<DT>(x.z, x.w));
}

template <int DT>
void sum_splits(const float* part, int splits, int64_t n, void* out0, void* out1, hipStream_t st) {
    attn_sum_kernel<DT><<<dim3((unsigned)((n / 4 + 255) / 256), out1 ? 2 : 1), 256, 0, st>>>(part, splits, n, out0, out1);
}

template <int DT, int DC, int MASK>
void launch(const AttnArgs& a, hipStream_t st) {
    if constexpr (DC == 64) {
        if (a.Tq && a.Tk && a.Tq <= kHeld && a.Tk <= kHeld && a.splits_kv == 1) {
            attn_dkv_kernel<DT, DC, MASK, true><<<(unsigned)(a.B * a.H), kThr, 0, st>>>(a);
            return;
        }
    }
    if (a.Tq) {
        attn_dq_kernel<DT, DC, MASK><<<(unsigned)((a.Tq + kHeld - 1) / kHeld * a.B * a.Hq * a.splits), kThr, 0, st>>>(a);
        if (a.splits > 1) sum_splits<DT>(a.part, a.splits, (int64_t)a.B * a.Tq * a.Hq * a.D, a.dq, nullptr, st);
    }
    if (a.Tk) {
        attn_dkv_kernel<DT, DC, MASK, false><<<(unsigned)((a.Tk + kHeld - 1) / kHeld * a.B * a.H * a.splits_kv), kThr, 0, st>>>(a);
        if (a.splits_kv > 1)
            sum_splits<DT>(a.part_kv, a.splits_kv, (int64_t)a.B * a.Tk * a.H * a.D, a.dk, a.dv, st);
    }
}

template <int DT, int DC>
void pick(const AttnArgs& a, hipStream_t st) {
    if (!a.mask) launch<DT, DC, kNoMask>(a, st);
    else if (a.ms[2] == 0) a.mask_type < 0 ? launch<DT, DC, kKeyMask>(a, st) : launch<DT, DC, kKeyAdd>(a, st);
    else launch<DT, DC, kFullMask>(a, st);
}

template <int DT>
void dispatch(const AttnArgs& a, hipStream_t st) {
    if (a.D <= 64) pick<DT, 64>(a, st);
    else if (a.D <= 80) pick<DT, 80>(a, st);
    else if (a.D <= 96) pick<DT, 96>(a, st);
    else pick<DT, 128>(a, st);
}

}  // namespace

int attention_backward(const AttnArgs& a, int dtype, hipStream_t st) {
    if (dtype == AXS6_F32) dispatch<AXS6_F32>(a, st);
    else if (dtype == AXS6_BF16) dispatch<AXS6_BF16>(a, st);
    else dispatch<AXS6_F16>(a, st);
    return AXS6_OK;
}

}  // namespace axs6
