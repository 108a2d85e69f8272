// Attention forward: o = softmax(scale q k^T + mask) v, heads of queries in
// groups that share a key head.
//
// With x_ij = scale q_i . k_j (and the mask), one pass over the keys keeps a
// row's running maximum m and sum l = sum_j exp(x_ij - m) and rescales the
// output when m grows; at the end o = sum_j exp(x_ij - m) v_j / l and
// m and log l, from which the backward makes a row's probabilities again.  A row that
// sees no key gives 0.
//
// Bound by the matrix cores (4 D operations a pair) and the exponentials
// beside them.  A wave holds 32 queries in registers; S^T = K q^T puts a
// query's scores in one lane and the lane 32 further on, so maximum and sum
// take one exchange, and the probabilities are the second product's operand
// in place.  The waves of a workgroup share the keys' tiles, which go from
// memory into the other of two LDS buffers while one is computed on: one
// barrier a tile.  Two waves a SIMD (at most 256 registers each) let one
// multiply while the other exponentiates: 1 x 16384, 16 heads of 128, causal,
// bf16: 1816 us with one, 1063 with two (2179 through registers with two
// barriers), 985 to 1018 with 128 keys a tile and 256 queries a workgroup,
// 1080 to 1116 TFLOP/s, where a bf16 matrix product of 8192^3 reaches 1139 on this card.
// The row's reference is only raised when a score passes it by 2^8, so the
// output is hardly ever rescaled; the sum is taken of the probabilities as they
// are rounded for the product.
// Few rows against many keys: the keys are split over workgroups, whose sums a
// second launch joins (4 x 4 queries of 16 heads, 8000 keys: 165 -> 31 us).
#include "attention.h"
#include "split_join.h"

namespace axs6 {
namespace {

// Scores may grow this far (a factor of 2^8 of a probability) past a row's
// reference before the row is rescaled, which then hardly ever happens.
constexpr float kSlack = 8.0f;

// A row of a split's partial results.
__device__ __forceinline__ int64_t split_row(const AttnArgs& a, int split, int b, int hq, int q) {
    return (((int64_t)split * a.B + b) * a.Hq + hq) * a.Tq + q;
}

// A row's results from the keys k0 .. k1 - 1 that it sees, one by one.
template <int DT>
__device__ void forward_row(const AttnArgs& a, int b, int hq, int q, int k0, int k1, int split, int lane) {
    const int h = hq / a.G;
    const float c = a.scale * kLog2e;
    const Two qv = load_two<DT>(a.q, b * a.qs[0] + q * a.qs[1] + hq * a.qs[2], a.D, lane);
    Two o = {0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int key = k0; key < k1 && !all_nan(o, a.D, lane); ++key) {
        const float f = pair_term(a, b, hq, q, key);
        if (f == -INFINITY) continue;
        const Two v = load_two<DT>(a.v, b * a.vs[0] + key * a.vs[1] + h * a.vs[2], a.D, lane);
        const float x =
            __builtin_fmaf(dot(qv, load_two<DT>(a.k, b * a.ks[0] + key * a.ks[1] + h * a.ks[2], a.D, lane)), c, f);
        const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(x - ref);
        m = mn;
        l = l * alpha + p;
        o = {o.x * alpha + p * v.x, o.y * alpha + p * v.y};
    }
    if (a.splits > 1) {
        const int64_t at = split_row(a, split, b, hq, q);
        if (lane == 0) { a.stat[2 * at] = m; a.stat[2 * at + 1] = l; }
        store_two<AXS6_F32>(a.part, at * a.D, o, a.D, lane);
        return;
    }
    const float rl = l == 0.0f ? 0.0f : 1.0f / l;
    store_two<DT>(a.o, (((int64_t)b * a.Tq + q) * a.Hq + hq) * a.D, {o.x * rl, o.y * rl}, a.D, lane);
    if (a.stats && lane == 0) a.stats[((int64_t)b * a.Hq + hq) * a.Tq + q] = row_stats(m, l);
}

// The forms of the kernel: four waves; eight that hold twice the queries; two
// groups of four that hold the same queries and take every second tile of keys,
// for 16-bit problems of at most a workgroup a CU, which would leave half the
// waves out (2 x 1024, 16 heads of 128, causal: 28 -> 24 us; in float32, where
// the matrix cores take their time with either, 64 x 128 gets 15 -> 18).
enum Form { kFour, kEight, kPaired };

// Queries and keys of a workgroup's tile.
template <int DT, int DC, int FORM> struct FwdShape {
    static constexpr int kWaves = FORM == kEight ? 8 : 4;   // of a group
    static constexpr int kGroups = FORM == kPaired ? 2 : 1;
    static constexpr int kKeys = DT == AXS6_F32 ? 64 : FORM == kEight || DC <= 64 ? 128 : 64;
    static constexpr int kQ = 32 * kWaves, kThreads = 64 * kWaves * kGroups;
    // two waves a SIMD, of which one computes softmax while the other multiplies
    static constexpr int kOccupancy = DT == AXS6_F32 ? 1 : 2;
};

template <int DT, int DC, int MASK, int FORM>
__global__ __launch_bounds__((FwdShape<DT, DC, FORM>::kThreads), (FwdShape<DT, DC, FORM>::kOccupancy)) void
attn_fwd_kernel(AttnArgs a) {
    using T = Tile<DT, DC>;
    using S = FwdShape<DT, DC, FORM>;
    constexpr int NK = S::kKeys / 32, W = S::kWaves, GROUPS = S::kGroups;
    // keys, then values; of each group two buffers
    __shared__ __attribute__((aligned(1024))) char kv[2][GROUPS][2][S::kKeys * T::kPitch];
    __shared__ __attribute__((aligned(16))) float terms[GROUPS][2][MASK == kKeyMask ? S::kKeys : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = wave % W, group = wave / W, tid = threadIdx.x % (64 * W);
    auto& kt = kv[0][group];
    auto& vt = kv[1][group];
    auto& term = terms[group];
    const int q_tiles = (a.Tq + S::kQ - 1) / S::kQ;
    int bh, piece;
    work_item(blockIdx.x, a.B * a.Hq, q_tiles * a.splits, a.causal, bh, piece);
    const int b = bh / a.Hq, hq = bh % a.Hq, h = hq / a.G, split = piece % a.splits;
    const int q0 = (q_tiles - 1 - piece / a.splits) * S::kQ;   // a causal mask's longest rows first
    const int off = a.Tk - a.Tq;
    const int q_last = q0 + S::kQ < a.Tq ? q0 + S::kQ - 1 : a.Tq - 1;
    int keys = a.causal ? q_last + off + 1 : a.Tk;
    keys = keys < 0 ? 0 : keys > a.Tk ? a.Tk : keys;
    int first = 0, tiles = (keys + S::kKeys - 1) / S::kKeys;
    if (a.splits > 1) {   // this workgroup's part of the keys
        const int per = (tiles + a.splits - 1) / a.splits;
        first = split * per < tiles ? split * per : tiles;
        tiles = first + per < tiles ? first + per : tiles;
    }
    // tiles whose every key every row of the workgroup sees, but for the mask
    const int free_keys = a.causal ? q0 + off + 1 : a.Tk;
    const int free_tiles = free_keys <= 0 ? 0 : (free_keys < a.Tk ? free_keys : a.Tk) / S::kKeys;

    const char* kb = reinterpret_cast<const char*>(a.k) + (b * a.ks[0] + h * a.ks[2]) * T::kBytes;
    const char* vb = reinterpret_cast<const char*>(a.v) + (b * a.vs[0] + h * a.vs[2]) * T::kBytes;
    Direct<DT, DC, S::kKeys, W> dk, dv;
    dk.init(a.ks[1], a.D, lane, w);
    dv.init(a.vs[1], a.D, lane, w);
    // the mask's term of key tid of tile t
    auto key_term = [&](int t) {
        const int key = t * S::kKeys + tid;
        return tid < S::kKeys && key < a.Tk ? mask_term(a, mask_row(a, b, hq, 0), key) : -INFINITY;
    };
    if (first + group < tiles) {
        const int t = first + group;
        dk.load(kt[0], kb, t * S::kKeys, a.Tk, a.D, w);
        dv.load(vt[0], vb, t * S::kKeys, a.Tk, a.D, w);
        if constexpr (MASK == kKeyMask) {
            const float f = key_term(t);
            if (tid < S::kKeys) term[0][tid] = f;
        }
    }
    const int q = q0 + 32 * w + (lane & 31), qr = q < a.Tq ? q : a.Tq - 1;
    const int limit = a.causal && qr + off + 1 < a.Tk ? qr + off + 1 : a.Tk;   // keys that the lane's row sees
    const char* mrow = MASK == kFullMask ? mask_row(a, b, hq, qr) : nullptr;
    u32x4 qf[T::kSteps];
    load_rows<DT, DC>(qf, a.q, b * a.qs[0] + qr * a.qs[1] + hq * a.qs[2], a.D, lane);
    f32x16 o[T::kResults];
#pragma unroll
    for (int d = 0; d < T::kResults; ++d) o[d] = zero16();
    float m = -INFINITY, l = 0.0f;   // the reference that scores are taken from; the sum of exponentials
    const float c = a.scale * kLog2e;

    const bool rows_here = q0 + 32 * w < a.Tq;   // the others only help to load
    const int w_last = q0 + 32 * w + 31 < a.Tq ? q0 + 32 * w + 31 : a.Tq - 1;   // the wave's last row and its keys
    const int w_keys = a.causal && w_last + off + 1 < a.Tk ? w_last + off + 1 : a.Tk;
    int buf = 0;
    for (int t = first + group; t - group < tiles; t += GROUPS, buf ^= 1) {
        tile_barrier();   // tile t is there, and nobody reads the other buffers any more
        float next_term = 0.0f;
        if (t + GROUPS < tiles) {
            dk.load(kt[buf ^ 1], kb, (t + GROUPS) * S::kKeys, a.Tk, a.D, w);
            dv.load(vt[buf ^ 1], vb, (t + GROUPS) * S::kKeys, a.Tk, a.D, w);
            if constexpr (MASK == kKeyMask) next_term = key_term(t + GROUPS);
        }
        const char *ks = kt[buf], *vs = vt[buf];
        const int k0 = t * S::kKeys;
        // A tile that the mask hides is passed over, and in float32 the 32 keys that
        // none of the wave's rows sees; in the 16-bit types those branches cost more
        // than they save (1 x 16384 forward 985 -> 1019 us).
        const int live = DT == AXS6_F32 && t >= free_tiles ? (w_keys - k0 + 31) >> 5 : NK;
        bool any = rows_here && (GROUPS == 1 || t < tiles) && (DT != AXS6_F32 || live > 0);
        bool plain = MASK == kNoMask;   // the mask adds nothing to any of the tile's scores
        if constexpr (MASK == kKeyMask) {
            const float f = term[buf][lane & (S::kKeys - 1)], g = S::kKeys > 64 ? term[buf][lane + S::kKeys - 64] : f;
            any = any && __any(!(f == -INFINITY && g == -INFINITY));
            plain = __all(f == 0.0f && g == 0.0f);
        }
        const float cs = plain ? c : 1.0f;   // what takes the scores to units of log2
        if (any) {
            f32x16 s[NK];
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                s[j] = zero16();
                if (DT == AXS6_F32 && j >= live) continue;
#pragma unroll
                for (int i = 0; i < T::kSteps; ++i) s[j] = mma<DT>(T::rows(ks, 32 * j, i, lane), qf[i], s[j]);
            }
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < NK; ++j)
                apply_mask<MASK>(a, s[j], c, k0 + 32 * j, &term[buf][MASK == kKeyMask ? 32 * j : 0], mrow, plain,
                                 t >= free_tiles, limit, lane);
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[j][i]);
            mx *= cs;
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (__any(mx > m + kSlack)) {   // m is -inf until the row sees a key
                const float mn = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < T::kResults; ++d) o[d] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            u32x4 pf[NK][2];
#pragma unroll
            for (int j = 0; j < NK; ++j) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], cs, -ref));
                fragments<DT>(s[j], pf[j]);
                if constexpr (DT == AXS6_F32) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) l += s[j][i];
                } else {   // the values as the product takes them
                    l = add_fragment<DT>(pf[j][0], l);
                    l = add_fragment<DT>(pf[j][1], l);
                }
            }
            if constexpr (DT == AXS6_F32) {
#pragma unroll
                for (int j = 0; j < NK; ++j)
                    if (j < live) T::accumulate(vs, 32 * j, s[j], pf[j], o, lane);
            } else {
#pragma unroll
                for (int d = 0; d < T::kResults; ++d)
#pragma unroll
                    for (int j = 0; j < 2 * NK; ++j)
                        o[d] = mma<DT>(T::col_fragment(vs, 16 * j, d, lane), pf[j / 2][j % 2], o[d]);
            }
        }
        if constexpr (MASK == kKeyMask)
            if (tid < S::kKeys) term[buf ^ 1][tid] = next_term;
    }
    l += __shfl_xor(l, 32, 64);
    if constexpr (GROUPS == 2) {   // one reference for both groups, then their sums
        __shared__ float other[2][2][W][32];
        if (lane < 32) { other[0][group][w][lane] = m; other[1][group][w][lane] = l; }
        __syncthreads();
        const float mo = other[0][group ^ 1][w][lane & 31], lo = other[1][group ^ 1][w][lane & 31];
        const float mn = fmaxf(m, mo), ref = mn == -INFINITY ? 0.0f : mn, f = __builtin_amdgcn_exp2f(m - ref);
        l = l * f + lo * __builtin_amdgcn_exp2f(mo - ref);
        m = mn;
#pragma unroll
        for (int d = 0; d < T::kResults; ++d) o[d] *= f;
        add_groups(o, reinterpret_cast<float*>(kv), group, w, lane);
        if (group == 1) return;
    }
    const bool bad = not_finite(o);
    if (q < a.Tq) {
        if (a.splits > 1) {
            const int64_t at = split_row(a, split, b, hq, q);
            if (lane < 32) { a.stat[2 * at] = m; a.stat[2 * at + 1] = l; }
            T::template store<AXS6_F32>(a.part, at * a.D, o, 1.0f, a.D, lane);
        } else {
            const float rl = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t row = (((int64_t)b * a.Tq + q) * a.Hq + hq) * a.D;
            T::template store<DT>(a.o, row, o, rl, a.D, lane);
            if (a.stats && lane < 32) a.stats[((int64_t)b * a.Hq + hq) * a.Tq + q] = row_stats(m, l);
        }
    }
    for (uint64_t rows = __ballot(bad && lane < 32 && q < a.Tq); rows; rows &= rows - 1)
        forward_row<DT>(a, b, hq, q0 + 32 * w + __builtin_ctzll(rows), first * S::kKeys,
                        tiles * S::kKeys < a.Tk ? tiles * S::kKeys : a.Tk, split, lane);
}

// FEW: at most kFewSplits, a thread four values; else a workgroup a row.
template <int DT, bool FEW>
__global__ __launch_bounds__(kJoinThreads) void attn_join_kernel(AttnArgs a) {
    using E = Elem<DT>;
    const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
    int64_t row = blockIdx.x;
    Joined j;
    if constexpr (FEW)
        j = join_few(a.part, a.stat, rows, (int64_t)blockIdx.x * kJoinThreads + threadIdx.x, a.splits, a.D, row);
    else
        j = join_row(a.part, a.stat, rows, row, a.splits, a.D);
    if (j.d < 0) return;
    const int64_t bh = row / a.Tq;
    const int q = (int)(row - bh * a.Tq);
    if (a.stats && j.d == 0) a.stats[row] = row_stats(j.m, j.l);
    const float rl = j.l == 0.0f ? 0.0f : 1.0f / j.l;
    auto* out = reinterpret_cast<typename E::S*>(a.o) + (((bh / a.Hq) * a.Tq + q) * a.Hq + bh % a.Hq) * a.D + j.d;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = E::from_f(j.o[i] * rl);
}

template <int DT>
void join(const AttnArgs& a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
    if (a.splits == 1) return;
    if (!join_by_value(rows, a.splits))
        attn_join_kernel<DT, false><<<(unsigned)rows, kJoinThreads, 0, st>>>(a);
    else
        attn_join_kernel<DT, true><<<(unsigned)((rows * (a.D / 4) + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, st>>>(a);
}

template <int DT, int DC, int MASK, int FORM>
void launch(const AttnArgs& a, hipStream_t st) {
    using S = FwdShape<DT, DC, FORM>;
    const unsigned grid = (unsigned)((a.Tq + S::kQ - 1) / S::kQ * a.B * a.Hq * a.splits);
    attn_fwd_kernel<DT, DC, MASK, FORM><<<grid, S::kThreads, 0, st>>>(a);
    join<DT>(a, st);
}

template <int DT, int DC>
void pick(const AttnArgs& a, hipStream_t st) {
    if constexpr (DT != AXS6_F32) {
        if ((int64_t)((a.Tq + 127) / 128) * a.B * a.Hq * a.splits <= 256 && (!a.mask || a.ms[2] == 0) &&
            a.Tk / a.splits > FwdShape<DT, DC, kPaired>::kKeys)
            return a.mask ? launch<DT, DC, kKeyMask, kPaired>(a, st) : launch<DT, DC, kNoMask, kPaired>(a, st);
    }
    if (a.mask) return a.ms[2] == 0 ? launch<DT, DC, kKeyMask, kFour>(a, st) : launch<DT, DC, kFullMask, kFour>(a, st);
    if constexpr (DT != AXS6_F32 && DC > 64) {
        // 256 queries a workgroup and 128 keys a tile from two workgroups a CU on:
        // fewer barriers (1 x 16384, 16 heads of 128, causal 990 us against 1063,
        // 2 x 4096 x 32 heads 333 against 327, without the mask 526 against 562)
        if ((int64_t)((a.Tq + 255) / 256) * a.B * a.Hq >= 512) return launch<DT, DC, kNoMask, kEight>(a, st);
    }
    launch<DT, DC, kNoMask, kFour>(a, st);
}

template <int DT>
void dispatch(const AttnArgs& a, hipStream_t st) {
    if (a.D <= 64) pick<DT, 64>(a, st);
    else if (a.D <= 80) pick<DT, 80>(a, st);
    else if (a.D <= 96) pick<DT, 96>(a, st);
    else pick<DT, 128>(a, st);
}

// Parts that an axis of `steps` tiles is split in, so that `groups` workgroups
// become `want`, of `least` tiles each at the least.
int split_count(int64_t groups, int64_t steps, int64_t want, int64_t least, int64_t most) {
    if (groups <= 0) return 1;
    int64_t s = (want + groups - 1) / groups;
    s = s < steps / least ? s : steps / least;
    s = s < most ? s : most;
    return s < 1 ? 1 : (int)s;
}

// Few rows against many keys: the keys are split until the 256 CUs have work,
// 256 keys a part at the least.
int forward_splits(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq) {
    const int64_t groups = (Tq + 127) / 128 * B * Hq;
    return groups >= 256 ? 1 : split_count(groups, Tk / 256, 512, 1, kMaxSplits);
}
// The backward walks over keys for dq, as the forward, and over the queries of a
// group's heads for dk and dv.  There a causal mask gives some keys' workgroups
// far more queries than others': four workgroups for each place on the chip's
// CUs even that out, where two fill it.
int key_splits(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t H, bool causal) {
    return split_count((Tk + 127) / 128 * B * H, (Tq + 31) / 32 * (H ? Hq / H : 1), causal ? 1024 : 512, 8, 16);
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
    // a tile's rows are addressed by 32-bit byte offsets from its first
    if (strides[1] < 0 || strides[1] >= AXS6_ATTENTION_MAX_TOKEN_STRIDE)
        return fail(AXS6_ERR_UNSUPPORTED, "%s: the tokens of %s are not 0 to %d elements apart", fn, name,
                    AXS6_ATTENTION_MAX_TOKEN_STRIDE - 1);
    return AXS6_OK;
}

int scratch(const char* fn, const void* workspace, int64_t bytes, int64_t need) {
    if (need && (!workspace || bytes < need || (uintptr_t)workspace % 16))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld bytes required, got %lld", fn,
                    (long long)need, (long long)bytes);
    return AXS6_OK;
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int64_t axs6_attention_forward_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t D) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || Hq <= 0 || D <= 0) return 0;
    const int64_t s = forward_splits(B, Tq, Tk, Hq);
    return s == 1 ? 0 : s * B * Hq * Tq * (D + 2) * (int64_t)sizeof(float);
}

extern "C" int64_t axs6_attention_backward_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t H, int64_t D,
                                                     int32_t causal) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || Hq <= 0 || H <= 0 || D <= 0) return 0;
    const int64_t s = forward_splits(B, Tq, Tk, Hq), kv = key_splits(B, Tq, Tk, Hq, H, causal);
    return ((s == 1 ? 0 : s * B * Tq * Hq * D) + (kv == 1 ? 0 : 2 * kv * B * Tk * H * D)) * (int64_t)sizeof(float) +
           B * Hq * ((Tq + 31) / 32) * (int64_t)sizeof(float2);
}

extern "C" int axs6_attention_forward(const void* q, const void* k, const void* v, int32_t dtype, int64_t B, int64_t Tq,
                                      int64_t Tk, int64_t Hq, int64_t H, int64_t D, const int64_t* q_strides,
                                      const int64_t* k_strides, const int64_t* v_strides, const void* mask,
                                      int32_t mask_type, const int64_t* mask_strides, int32_t causal, float scale,
                                      void* out, float* stats, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "axs6_attention_forward";
    AttnArgs a{};
    int rc = fill(fn, a, dtype, B, Tq, Tk, Hq, H, D, mask, mask_type, mask_strides, causal, scale);
    if (rc) return rc;
    if (B * Tq * Hq == 0) return AXS6_OK;
    if ((rc = operand(fn, "q", q, q_strides, dtype, a.qs))) return rc;
    if (Tk && ((rc = operand(fn, "k", k, k_strides, dtype, a.ks)) || (rc = operand(fn, "v", v, v_strides, dtype, a.vs))))
        return rc;
    if (!out || (uintptr_t)out % 16) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: output null or not aligned", fn);
    if ((uintptr_t)stats % 8) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: stats not aligned to 8 bytes", fn);
    a.q = q; a.k = k; a.v = v; a.o = out; a.stats = reinterpret_cast<float2*>(stats);
    a.splits = forward_splits(B, Tq, Tk, Hq);
    const int64_t need = axs6_attention_forward_workspace(B, Tq, Tk, Hq, D);
    if ((rc = scratch(fn, workspace, workspace_bytes, need))) return rc;
    a.part = reinterpret_cast<float*>(workspace);
    a.stat = a.part + a.splits * B * Hq * Tq * D;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AXS6_F32) dispatch<AXS6_F32>(a, st);
    else if (dtype == AXS6_BF16) dispatch<AXS6_BF16>(a, st);
    else dispatch<AXS6_F16>(a, st);
    return check_launch(fn);
}

extern "C" int axs6_attention_backward(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                       const float* stats, int32_t dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
                                       int64_t H, int64_t D, const int64_t* dout_strides, const int64_t* q_strides,
                                       const int64_t* k_strides, const int64_t* v_strides, const void* mask,
                                       int32_t mask_type, const int64_t* mask_strides, int32_t causal, float scale,
                                       float* delta, void* dq, void* dk, void* dv, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
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
    if ((Tq && (!stats || !delta || !dq)) || (Tk && (!dk || !dv)))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null stats, delta or gradient", fn);
    if ((uintptr_t)stats % 8) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: stats not aligned to 8 bytes", fn);
    if ((uintptr_t)dq % 16 || (uintptr_t)dk % 16 || (uintptr_t)dv % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: gradients not aligned to 16 bytes", fn);
    a.q = q; a.k = k; a.v = v; a.out = out; a.dout = dout; a.delta = delta;
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
    a.dq = dq; a.dk = dk; a.dv = dv;
    a.splits = forward_splits(B, Tq, Tk, Hq);
    a.splits_kv = key_splits(B, Tq, Tk, Hq, H, causal);
    if ((rc = scratch(fn, workspace, workspace_bytes, axs6_attention_backward_workspace(B, Tq, Tk, Hq, H, D, causal))))
        return rc;
    a.part = reinterpret_cast<float*>(workspace);
    a.part_kv = a.part + (a.splits == 1 ? 0 : a.splits * B * Tq * Hq * D);
    a.bounds = reinterpret_cast<float2*>(a.part_kv + (a.splits_kv == 1 ? 0 : 2 * a.splits_kv * B * Tk * H * D));
    attention_backward(a, dtype, (hipStream_t)stream);
    return check_launch(fn);
}
