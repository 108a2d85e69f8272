// Attention of the newest tokens over the 8-bit cache (generation).
//
// Sequence b holds n_b tokens, the last Tq of which are the queries: query t
// of head h sees keys j <= n_b - Tq + t of the key head h / G, G = Hq / Hkv:
//   x_j = scale * ks * (q . kc_j),  o = sum_j softmax(x)_j vs * vc_j
// with codes kc, vc and the block's scales ks, vs.  A query that sees nothing
// gives 0.
//
// Bound by HBM: each code is read once, 2 D bytes a token and key head, for
// all G * Tq rows that share them.  The products run on the matrix cores in
// f16, where the codes are exact (|code| <= 127): a query row is scaled by a
// power of two to [128, 256) and rounded to f16 (bf16 and f16 queries exactly,
// but for values 2^-21 below the row's largest), a float32 query split in two
// f16 terms (22 bits); probabilities go in as f16 times 2^14 (11 bits; for
// float32 in two terms), so that one of 2^-28 of the largest still counts.
// Maximum, sums and outputs are float32.
//
// S^T = K q^T by 16x16x32 instructions with the keys as rows: a lane then
// holds 8 consecutive keys of one query row, which is the order in which the
// second product takes them, so the probabilities never leave their registers.
// A workgroup's waves take every so-many-th block of its range; where there are
// few rows the blocks are split over more workgroups and joined by a second
// launch, in which a thread takes one split's factor and groups of threads every
// so-many-th sum (one wave a row that walked over the splits took three times the
// attention: 1 x 16384 tokens, 8 key heads for 32, 48 us against 15).
// Measured: 64 sequences of 4096 to 16383 tokens, 8 key heads of 128 for 64,
// 290 us, 4.6 TB/s (a copy of 4 GiB runs at 4.7 on this card); one of 131072
// 55 us; one of 300, where launches and latency count, 8.7 us.  A prompt's workgroups
// each read and convert all the blocks before them again: 1024 tokens, 8 key heads of
// 128 for 32, 58 us, 4096 453 us.  Holding the next
// block's codes on their way costs registers and with them waves: 64 x 2048
// tokens 22.8 -> 25.7 us.
#include <math.h>

#include "axs6_internal.h"
#include "kv_cache.h"
#include "nf5_device.h"
#include "split_join.h"

namespace axs6 {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kProbScale = 16384.0f;   // 2^14
constexpr float kSumScale = 1048576.0f;  // 2^20: sums are held as 2^-20 of themselves, so that values near
                                         // float32's largest, summed before they are divided, stay finite

struct KvAttnArgs {
    const void* q;
    int64_t qs[3];            // batch, token, head, in elements
    const int8_t *kc, *vc;
    const float *ks, *vs;
    const int64_t* lengths;
    void* out;                // (B, Tq, Hq, D) contiguous
    float *part, *stat;       // of each split and row: the sums of D values; maximum and sum
    int64_t rows_all;         // B * H * rows
    int H, G, Tq, D, nb, rows, row_tiles, splits;
    int qvec;
    float scale;
};

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

// Sixteen values of a query from element i.
template <int DT>
__device__ __forceinline__ void load16(const void* p, int64_t i, bool vec, float* f) {
    using E = Elem<DT>;
    const auto* q = reinterpret_cast<const typename E::S*>(p) + i;
    if (vec) {
#pragma unroll
        for (int j = 0; j < 16; j += E::V) E::unpack(*reinterpret_cast<const u32x4*>(q + j), f + j);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = E::to_f(q[j]);
    }
}

// A block's codes as a lane takes them.
template <int NC>
__device__ __forceinline__ void load_block(u32x4 (&k)[2][NC], uint2 (&v)[NC * 4], const KvAttnArgs& a, int64_t cell,
                                           int n16, int g4) {
    const int8_t* kc = a.kc + cell * kKvBlock * a.D;
    const int8_t* vc = a.vc + cell * kKvBlock * a.D;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            k[tt][c] = u32x4{0, 0, 0, 0};
            const int key = 8 * (n16 >> 2) + 4 * tt + (n16 & 3);
            if (64 * c + 16 * g4 < a.D)
                k[tt][c] = *reinterpret_cast<const u32x4*>(kc + key * a.D + 64 * c + 16 * g4);
        }
#pragma unroll
    for (int d = 0; d < NC * 4; ++d) {
        v[d] = make_uint2(0, 0);
        if (16 * d < a.D) v[d] = *reinterpret_cast<const uint2*>(vc + (16 * d + n16) * kKvBlock + 8 * g4);
    }
}

// NC: 64-value pieces of a head.  NR: 16-row pieces of queries that a wave takes
// against each block.  WAVES: of a workgroup, each of which takes every WAVES-th
// block of its range.
template <int DT, int NC, int NR, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void kv_attention_kernel(KvAttnArgs a) {
    constexpr int TERMS = DT == AXS6_F32 ? 2 : 1;
    constexpr int ND = NC * 4;   // 16-value pieces of a head
    __shared__ float sh_o[WAVES / 2][NR * ND * 4][64];
    __shared__ float sh_m[WAVES][NR * 16], sh_l[WAVES][NR * 16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n16 = lane & 15, g4 = lane >> 4;
    const int rt = blockIdx.x % a.row_tiles, bh = blockIdx.x / a.row_tiles, h = bh % a.H, b = bh / a.H;
    const int64_t cap = (int64_t)a.nb * kKvBlock;
    int64_t len = a.lengths[b];
    len = len < 0 ? 0 : len > cap ? cap : len;
    const int r0 = rt * NR * 16, r_top = r0 + NR * 16 < a.rows ? r0 + NR * 16 - 1 : a.rows - 1;
    const int keys = (int)(len - a.Tq) + r_top / a.G + 1;
    const int blocks = keys <= 0 ? 0 : (keys + kKvBlock - 1) / kKvBlock;
    const int per = (blocks + a.splits - 1) / a.splits;
    const int b0 = blockIdx.y * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    const int64_t cell0 = (int64_t)bh * a.nb;
    u32x4 kr[2][NC];
    uint2 vr[ND];
    if (b0 + w < b1) load_block<NC>(kr, vr, a, cell0 + b0 + w, n16, g4);

    // the rows' queries, scaled, in the products' order: piece c, value 16 g4 + j
    f16x8 qf[NR][TERMS][NC][2];
    float rs[NR];
    int last[NR];   // the last key that the lane's row sees
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int r = r0 + 16 * n + n16, rr = r < a.rows ? r : a.rows - 1, t = rr / a.G, hq = h * a.G + rr % a.G;
        last[n] = (int)(len - a.Tq) + t;
        float f[NC][16], amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < 16; ++j) f[c][j] = 0.0f;
            if (64 * c + 16 * g4 < a.D)
                load16<DT>(a.q, b * a.qs[0] + t * a.qs[1] + hq * a.qs[2] + 64 * c + 16 * g4, a.qvec, f[c]);
#pragma unroll
            for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(f[c][j]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
        amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
        const int e = amax > 0.0f && isfinite(amax) ? ilogbf(amax) - 7 : 0;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float x = ldexpf(f[c][j], -e);
                const _Float16 hi = (_Float16)x;
                qf[n][0][c][j >> 3][j & 7] = hi;
                if constexpr (TERMS == 2) qf[n][1][c][j >> 3][j & 7] = (_Float16)(x - (float)hi);
            }
        rs[n] = ldexpf(a.scale * kLog2e, e);
    }

    f32x4 o[NR][ND];
    float m[NR], l[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int d = 0; d < ND; ++d) o[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    for (int blk = b0 + w; blk < b1; blk += WAVES) {
        const int64_t cell = cell0 + blk;
        if (blk != b0 + w) load_block<NC>(kr, vr, a, cell, n16, g4);   // the first came before the queries
        const float ks = a.ks[cell], vs = a.vs[cell] * (1.0f / kProbScale);   // the codes bring 1 / kSumScale
        f32x4 s[NR][2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
            for (int n = 0; n < NR; ++n) s[n][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const f16x8 k0 = codes_f16<false>(kr[tt][c].x, kr[tt][c].y), k1 = codes_f16<false>(kr[tt][c].z, kr[tt][c].w);
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int u = 0; u < TERMS; ++u) {
                        s[n][tt] = mma(k0, qf[n][u][c][0], s[n][tt]);
                        s[n][tt] = mma(k1, qf[n][u][c][1], s[n][tt]);
                    }
            }
        }
        f16x8 pf[NR][TERMS];
        float alpha[NR], vsn[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            // a row that sees none of the block takes nothing of it, whatever its scale
            vsn[n] = blk * kKvBlock > last[n] ? 0.0f : vs;
            float x[8], mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = blk * kKvBlock + 8 * g4 + j <= last[n] ? s[n][j >> 2][j & 3] * (rs[n] * ks) : -INFINITY;
                mx = fmaxf(mx, x[j]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float mn = fmaxf(m[n], mx), ref = mn == -INFINITY ? 0.0f : mn;
            alpha[n] = __builtin_amdgcn_exp2f(m[n] - ref);
            m[n] = mn;
            l[n] *= alpha[n];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = __builtin_amdgcn_exp2f(x[j] - ref);
                l[n] += p;
                const float y = p * kProbScale;
                pf[n][0][j] = (_Float16)y;
                if constexpr (TERMS == 2) pf[n][1][j] = (_Float16)(y - (float)pf[n][0][j]);
            }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (16 * d >= a.D) continue;
            const f16x8 vf = codes_f16<true>(vr[d].x, vr[d].y);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < TERMS; ++u) y = mma(vf, pf[n][u], y);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][d][i] = o[n][d][i] * alpha[n] + y[i] * vsn[n];
            }
        }
    }
    // join the waves: the four lanes of a row, then the upper half of the waves
    // into the lower, and again
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        l[n] += __shfl_xor(l[n], 16, 64);
        l[n] += __shfl_xor(l[n], 32, 64);
        if (g4 == 0) { sh_m[w][16 * n + n16] = m[n]; sh_l[w][16 * n + n16] = l[n]; }
    }
    __syncthreads();
    float lt[NR], mt[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        mt[n] = sh_m[0][16 * n + n16];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) mt[n] = fmaxf(mt[n], sh_m[i][16 * n + n16]);
        const float ref = mt[n] == -INFINITY ? 0.0f : mt[n];
        lt[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i)
            lt[n] += sh_l[i][16 * n + n16] * __builtin_amdgcn_exp2f(sh_m[i][16 * n + n16] - ref);
        const float f = __builtin_amdgcn_exp2f(m[n] - ref);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[n][d] *= f;
    }
#pragma unroll
    for (int step = WAVES / 2; step >= 1; step >>= 1) {
        if (w >= step && w < 2 * step)
#pragma unroll
            for (int i = 0; i < NR * ND * 4; ++i) sh_o[w - step][i][lane] = o[i / (ND * 4)][i / 4 % ND][i % 4];
        __syncthreads();
        if (w < step)
#pragma unroll
            for (int i = 0; i < NR * ND * 4; ++i) o[i / (ND * 4)][i / 4 % ND][i % 4] += sh_o[w][i][lane];
        __syncthreads();
    }
    if (w != 0) return;
    using E = Elem<DT>;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int r = r0 + 16 * n + n16, t = r / a.G, hq = h * a.G + r % a.G;
        if (r >= a.rows) continue;
        const int64_t row = (int64_t)bh * a.rows + r;
        if (a.splits > 1) {
            const int64_t at = blockIdx.y * a.rows_all + row;
            if (g4 == 0) { a.stat[2 * at] = mt[n]; a.stat[2 * at + 1] = lt[n]; }
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (16 * d < a.D) *reinterpret_cast<f32x4*>(a.part + at * a.D + 16 * d + 4 * g4) = o[n][d];
        } else {
            const float rl = lt[n] == 0.0f ? 0.0f : kSumScale / lt[n];
            auto* out =
                reinterpret_cast<typename E::S*>(a.out) + (((int64_t)b * a.Tq + t) * a.H * a.G + hq) * a.D + 4 * g4;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (16 * d < a.D)
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[16 * d + i] = E::from_f(o[n][d][i] * rl);
        }
    }
}

// FEW: at most kFewSplits, a thread four values; else a workgroup a row.
template <int DT, bool FEW>
__global__ __launch_bounds__(kJoinThreads) void kv_join_kernel(KvAttnArgs a) {
    using E = Elem<DT>;
    int64_t row = blockIdx.x;
    Joined j;
    if constexpr (FEW)
        j = join_few(a.part, a.stat, a.rows_all, (int64_t)blockIdx.x * kJoinThreads + threadIdx.x, a.splits, a.D, row);
    else
        j = join_row(a.part, a.stat, a.rows_all, row, a.splits, a.D);
    if (j.d < 0) return;
    const int64_t bh = row / a.rows;
    const int r = (int)(row - bh * a.rows), t = r / a.G, hq = (int)(bh % a.H) * a.G + r % a.G;
    const float rl = j.l == 0.0f ? 0.0f : kSumScale / j.l;
    auto* out = reinterpret_cast<typename E::S*>(a.out) + (((bh / a.H) * a.Tq + t) * a.H * a.G + hq) * a.D + j.d;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = E::from_f(j.o[i] * rl);
}

// How a call is laid out: 16-row pieces a wave takes, workgroups of 8 waves or 4,
// workgroups that share a set of rows.
constexpr int64_t kMaxPartial = (int64_t)64 << 20;   // bytes of partial sums that splits by length may take
struct Plan {
    int nr, waves, row_tiles, splits;
};
Plan plan(int64_t BH, int64_t rows, int64_t D, int64_t blocks) {
    Plan p;
    // Two pieces a wave spare reading and converting the codes again (16 sequences of
    // 40 rows: 66 -> 64 us); four leave one wave a SIMD (87 us).
    p.nr = rows <= 16 || D > 128 ? 1 : 2;
    p.row_tiles = (int)((rows + 16 * p.nr - 1) / (16 * p.nr));
    const int64_t groups = BH * p.row_tiles;
    // Few rows and at most 16 blocks: one workgroup of 8 waves, for a second launch
    // that joins splits costs more than it saves (1 x 300 tokens 9.0 us, split 11.3).
    p.waves = groups < 256 && blocks <= 16 && p.nr == 1 && D <= 128 ? 8 : 4;
    // Splits: two workgroups a CU, or 128 blocks each at the most, which evens out
    // sequences of unequal length (64 sequences to 16383 tokens: 2048 workgroups
    // 280 us, 1024 298; 1 x 131072: 512 workgroups 50 us, 1024 55).
    int64_t s = (512 + groups - 1) / (groups > 0 ? groups : 1), by_length = (blocks + 127) / 128;
    // The capacity is known here, the lengths are not: splits by it cost a prompt, whose rows
    // are many, most where it is short.  Their partial sums stay within 64 MiB, which
    // generation does not reach (1 x 4096 tokens, 32 heads on 8 of 128, a cache of 16384: 693 us
    // and 260 MiB of partial sums, now 453 and none).
    const int64_t bytes = BH * rows * (D + 2) * (int64_t)sizeof(float), most = kMaxPartial / (bytes > 0 ? bytes : 1);
    by_length = by_length < most ? by_length : most;
    s = s > by_length ? s : by_length;
    s = s < blocks / 4 ? s : blocks / 4;
    s = s < kMaxSplits ? s : kMaxSplits;
    p.splits = p.waves == 8 || s < 1 ? 1 : (int)s;
    return p;
}

template <int DT, int NC>
void launch_kernel(const KvAttnArgs& a, const Plan& p, int64_t B, hipStream_t st) {
    const dim3 grid((unsigned)(B * a.H * a.row_tiles), (unsigned)a.splits);
    if constexpr (NC <= 2) {
        if (p.waves == 8) {
            kv_attention_kernel<DT, NC, 1, 8><<<grid, 512, 0, st>>>(a);
            return;
        }
        if (p.nr == 2) {
            kv_attention_kernel<DT, NC, 2, 4><<<grid, 256, 0, st>>>(a);
            return;
        }
    }
    kv_attention_kernel<DT, NC, 1, 4><<<grid, 256, 0, st>>>(a);
}

template <int DT>
void launch_attention(const KvAttnArgs& a, const Plan& p, int64_t B, hipStream_t st) {
    switch ((a.D + 63) / 64) {
        case 1: launch_kernel<DT, 1>(a, p, B, st); break;
        case 2: launch_kernel<DT, 2>(a, p, B, st); break;
        case 3: launch_kernel<DT, 3>(a, p, B, st); break;
        default: launch_kernel<DT, 4>(a, p, B, st); break;
    }
    if (a.splits == 1) return;
    if (!join_by_value(a.rows_all, a.splits))
        kv_join_kernel<DT, false><<<(unsigned)a.rows_all, kJoinThreads, 0, st>>>(a);
    else
        kv_join_kernel<DT, true><<<(unsigned)((a.rows_all * (a.D / 4) + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int64_t axs6_kv_attention_workspace(int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D, int64_t blocks) {
    if (B <= 0 || Tq <= 0 || H <= 0 || Hq <= 0 || Hq % H || D <= 0 || blocks <= 0) return 0;
    const int64_t rows = Tq * (Hq / H), s = plan(B * H, rows, D, blocks).splits;
    return s == 1 ? 0 : s * B * H * rows * (D + 2) * (int64_t)sizeof(float);
}

extern "C" int axs6_kv_attention(const void* q, int32_t dtype, int64_t B, int64_t Tq, int64_t Hq, int64_t H, int64_t D,
                                 const int64_t* q_strides, const void* k_codes, const float* k_scales,
                                 const void* v_codes, const float* v_scales, int64_t blocks, const int64_t* lengths,
                                 float scale, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "axs6_kv_attention";
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    int rc = check_cache(fn, B, H, D, blocks, k_codes, k_scales, v_codes, v_scales);
    if (rc) return rc;
    if (Tq < 0 || Hq < 0 || (H > 0 && Hq % H))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: %lld query heads for %lld key heads", fn, (long long)Hq, (long long)H);
    if (!isfinite(scale)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: the scale must be finite", fn);
    if (B * Tq * Hq == 0) return AXS6_OK;
    if (H == 0 || blocks == 0) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: an empty cache", fn);
    if (!q || !q_strides || !lengths || !out) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null operand", fn);
    const int64_t es = dtype == AXS6_F32 ? 4 : 2, vl = 16 / es, rows = Tq * (Hq / H);
    if (rows > (1 << 24) || B * H * ((rows + 15) / 16) > ((int64_t)1 << 31) - 1 || B * H * rows > ((int64_t)1 << 31) - 1)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    if ((uintptr_t)q % es || (uintptr_t)out % es)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not element-aligned", fn);
    KvAttnArgs a{};
    a.q = q; a.kc = reinterpret_cast<const int8_t*>(k_codes); a.vc = reinterpret_cast<const int8_t*>(v_codes);
    a.ks = k_scales; a.vs = v_scales; a.lengths = lengths; a.out = out;
    a.qvec = (uintptr_t)q % 16 == 0;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = q_strides[i];
        a.qvec = a.qvec && q_strides[i] % vl == 0;
    }
    a.H = (int)H; a.G = (int)(Hq / H); a.Tq = (int)Tq; a.D = (int)D; a.nb = (int)blocks; a.rows = (int)rows;
    const Plan p = plan(B * H, rows, D, blocks);
    a.row_tiles = p.row_tiles; a.rows_all = B * H * rows; a.scale = scale; a.splits = p.splits;
    if (a.splits > 1) {
        const int64_t need = axs6_kv_attention_workspace(B, Tq, Hq, H, D, blocks);
        if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
            return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld bytes required, got %lld", fn,
                        (long long)need, (long long)workspace_bytes);
        a.part = reinterpret_cast<float*>(workspace);
        a.stat = a.part + a.splits * a.rows_all * D;
    }
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AXS6_F32) launch_attention<AXS6_F32>(a, p, B, st);
    else if (dtype == AXS6_BF16) launch_attention<AXS6_BF16>(a, p, B, st);
    else launch_attention<AXS6_F16>(a, p, B, st);
    return check_launch(fn);
}
