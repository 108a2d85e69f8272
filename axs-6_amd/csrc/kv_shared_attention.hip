// Attention of sequences that share a prefix, over the 8-bit cache.
//
// W sequences in a row continue one prefix.  Sequence b's tokens are the prefix's n_p and
// then the n_b of its own cache; query t (of Tq) stands at place n_p + n_b - Tq + t and
// sees the places up to its own:
//   x_j = scale * ks * (q . kc_j),  o = sum_j softmax(x)_j vs * vc_j
// over the keys of both caches (codes kc, vc, a block's scales ks, vs).  The prefix is read
// once for the rows of all W sequences, W Tq G of a key head.
//
// One launch for both, in which a workgroup takes 64 rows against a piece of the prefix,
// or a sequence's rows against its own blocks (those are bound by HBM, the prefix's with
// many rows by the matrix cores and the softmax: side by side each hides the other), and
// leaves maximum, sum and D sums a row; a second launch joins a row's pieces.  The prefixes'
// pieces are cut from all the blocks that they hold, so that workgroups have equal work
// whatever the lengths, which only the device knows.
//
// Products as in the cache attention (S^T = K q^T by 16x16x32 f16 instructions in which codes are exact, probabilities
// stay in their lanes).  A block's value scale goes into its probabilities' exponent, which counts from a reference of
// its own; the references move only when a score passes them by kSlack, and between that the sums stay where the products
// add to them.  Probabilities go in as f16 times 2^11 (float32: two terms): 11 bits down to 2^-25 of the largest, and some
// down to 2^-35 (the cache attention has 2^14, 2^-28 and 2^-38: its reference is the maximum itself).  Beside a bf16
// output's own rounding that does not count; f16 outputs are off by 2.7e-4 where their rounding alone makes 2.1e-4 (a second
// term for f16 too would make it that: 32000 tokens for 128 sequences 145 -> 172 us, 3 x 21 of 5 queries 37.7 -> 40.5).
// Turning codes into f16 costs as much as a block's softmax for 32 rows: a prefix's workgroup does it once for its four
// waves' 64 rows, into LDS; rows of one sequence are few, and there each wave has blocks of its own, whose codes come
// straight from memory into LDS.
//
// Measured (launch + join): a prefix of 32000 tokens for 128 sequences, 32 heads on 8 of 128, bf16, 131 + 9 us, 490
// TFLOP/s; 8 of 16383 for 8 sequences each, 64 heads on 8, 60 + 9, 3.1 TB/s; 3 of 7777 for 21 sequences of 5 queries, 12
// heads on 4 of 80, f16, 27.5 + 9.4; one of 300 for 4 sequences, f32, 8.8 + 4.8.  The join takes 9.3 us for 24 MB of sums as
// for 36: a chain of exponentials and rescaling over a row's 15 to 19 pieces.  At the first: vector instructions (150 a block
// and 16 rows, 40 of them for the codes) fill 60% of the time, LDS 46%, the matrix cores 23%, and waits for LDS and the
// others' part of a tile the rest.  16 rows a wave at four workgroups a CU against 32 rows, which read LDS half as often,
// at two: 140 us against 185.
#include "kv_attention.h"

namespace axs6 {
namespace {

typedef __attribute__((address_space(3))) void lds_void;

constexpr int kSharedWaves = 4, kSharedThreads = 64 * kSharedWaves;
constexpr float kSlack = 4.0f;          // in units of log2 (0: 32000 tokens for 128 sequences 148 -> 154 us, 2: 149)
// A maximum from which the products first become their distances from it: with the value scale's exponent added at once
// that would lose its digits (below, 1e-5 of a weight, of which f16 keeps 2^-12; float32's always do).
constexpr float kLarge = 256.0f;
constexpr int kWeightLog2 = 11;         // probabilities go in times 2^11; with 2^kSlack still an f16
constexpr int kSumLog2 = 20;            // sums go out divided by 2^20
// Prefixes whose blocks are shared out evenly, a lane of a wave each (four of 8000 tokens beside 60 of 300, 4 sequences
// each: 46 us, by prefix 115; 64 of 1000 50 and 45, for the even cut's own work is 1 us and more).
constexpr int kMaxEven = 64;

struct SharedArgs {
    const void* q;
    int64_t qs[3];                      // batch, token, head, in elements
    const int8_t *kc[2], *vc[2];        // the prefixes, the sequences' own
    const float *ks[2], *vs[2];
    const int64_t* lengths[2];
    void* out;                          // (B, Tq, Hq, D) contiguous
    float* part[2];                     // of each piece, head and row D sums; then (maximum, sum)
    float* stat[2];
    int P, W, H, G, Tq, D, qvec;
    int nb[2];                          // blocks
    int rows[2], row_tiles[2];          // of a head: W Tq G, Tq G
    int pieces[2];                      // of all prefixes; of each sequence
    int even;                           // whether the prefixes' pieces are cut from all their blocks
    int units, prefix_groups;           // (piece, head) of the prefixes; workgroups that take them
    float scale;
};

__device__ __forceinline__ int clamp_length(int64_t n, int nb) {
    const int64_t cap = (int64_t)nb * kKvBlock;
    return (int)(n < 0 ? 0 : n > cap ? cap : n);
}
__device__ __forceinline__ float lane_value(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
__device__ __forceinline__ int blocks_of(int n) { return (n + kKvBlock - 1) / kKvBlock; }

// The pieces of the prefixes.  Even: lane p < P <= 64 has prefix p; every piece is of `size`
// blocks but each prefix's last, size the smallest with which all pieces suffice.  Else a
// prefix has pieces / P of them.
struct Pieces {
    int blocks, size, first, count;   // the lane's prefix: blocks, of a piece, first piece, pieces
};
__device__ __forceinline__ Pieces even_pieces(const SharedArgs& a, int lane) {
    Pieces c;
    c.blocks = lane < a.P ? blocks_of(clamp_length(a.lengths[0][lane], a.nb[0])) : 0;
    int total = c.blocks;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o, 64);
    const int spare = a.pieces[0] - a.P + 1;   // a prefix's last piece may be short: P - 1 pieces more
    c.size = (total + spare - 1) / spare;
    c.size = c.size < 1 ? 1 : c.size;
    c.count = (c.blocks + c.size - 1) / c.size;
    c.first = c.count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(c.first, o, 64);
        if (lane >= o) c.first += x;
    }
    c.first -= c.count;
    return c;
}

// A head of up to 16 ND values in LDS: a block's key codes, 32 rows of kRow 16-byte pieces, and its value codes, 16 ND
// rows of two.
template <int ND> constexpr int kRow = ND <= 4 ? 4 : ND <= 8 ? 8 : 16;
template <int ND> constexpr int kKeyBytes = kKvBlock * kRow<ND> * 16;
template <int ND> constexpr int kSlotBytes = kKeyBytes<ND> + ND * 512;

// Piece j of key row r lies in place j ^ key_turn(r): the 16 rows that a fragment reads at one piece, 8 a + 4 tt + b, fall
// on all banks.  Of r = 64 i / kRow + lane / kRow it is key_turn(64 i / kRow) ^ key_turn(lane / kRow).
template <int ND> __device__ __forceinline__ constexpr int key_turn(int r) {
    constexpr int L = kRow<ND> == 4 ? 0 : kRow<ND> == 8 ? 1 : 2;
    return ((r >> 3) & 3) << L | (r & 3) >> (2 - L);
}

// A block's codes on their way to the wave's slot, 1 KB an instruction; what lies past the head's values arrives as
// zeros.  The two halves of a value's row change places in rows 8 .. 15 of 16.
template <int ND>
__device__ __forceinline__ void fetch_block(char* slot, const int8_t* kc, const int8_t* vc, int64_t cell, int D, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)   // the host pass knows no 16-byte form and would drop the kernel's stub
    const int bytes = kKvBlock * D;
    const auto kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(kc + cell * bytes), 0, bytes, 0x00020000);
    const auto vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(vc + cell * bytes), 0, bytes, 0x00020000);
    asm("" : "+v"(lane));   // the places are made again each time: as values kept over the loop they would cost registers
    const int row = lane / kRow<ND>, turned = lane % kRow<ND> ^ key_turn<ND>(row), at = row * D;
#pragma unroll
    for (int i = 0; i < kRow<ND> / 2; ++i) {
        const int j16 = (turned ^ key_turn<ND>(64 * i / kRow<ND>)) * 16;
        const int off = ND % 4 == 0 && D == 16 * kRow<ND> ? at + j16 : j16 < D ? at + j16 : bytes;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void*)(slot + i * 1024), 16, off, 64 * i / kRow<ND> * D, 0, 0);
    }
    const int half = (lane ^ ((lane >> 4) & 1)) * 16;
#pragma unroll
    for (int i = 0; i < ND / 2; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void*)(slot + kKeyBytes<ND> + i * 1024), 16, half, i * 1024, 0, 0);
#endif
}

// A wave's 16 NR rows (a lane has row 16 n + lane % 16) of a key head's: queries, what they see, and what attention
// leaves of the blocks so far.  l counts from the maximum m, o from the maximum w of x + log2(value scale) + unit.
// S 0: rows of all sequences of a prefix, 1: of one sequence.
template <int DT, int ND, int NR, int S>
struct Rows {
    static constexpr int TERMS = DT == AXS6_F32 ? 2 : 1;
    static constexpr int NC = (ND + 3) / 4;   // 64-value pieces of a head
    f16x8 qf[NR][TERMS][NC][2];
    float rs[NR];
    int last[NR];   // the last key that the lane's row sees
    int whole;      // keys that all the wave's rows see
    int unit;       // value scales count from 2^unit
    f32x4 o[NR][ND];
    float m[NR], w[NR], l[NR];

    // The queries from row r0 on, scaled to [128, 256): of piece c a lane has values 64 c + 16 g4 + j; HALVES: of both
    // its halves 8 g4 + j each.  `largest`: the largest value scale, the lanes' own yet.
    template <bool HALVES>
    __device__ __forceinline__ void init(const SharedArgs& a, int set, int h, int r0, int len, float largest, int lane) {
        const int n16 = lane & 15, g4 = lane >> 4, per_seq = a.Tq * a.G;
        whole = len;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            int r = r0 + 16 * n + n16;
            r = r < a.rows[S] ? r : a.rows[S] - 1;
            const int seq = S ? set : set * a.W + r / per_seq;
            r = S ? r : r % per_seq;
            const int t = r / a.G, hq = h * a.G + r % a.G;
            last[n] = len - a.Tq + t;
            if constexpr (S == 0) {   // the sequence's own tokens follow the prefix's
                const int64_t to = (int64_t)last[n] + clamp_length(a.lengths[1][seq], a.nb[1]);
                last[n] = (int)(to < len ? to : len - 1);
            }
            whole = last[n] + 1 < whole ? last[n] + 1 : whole;
            const int64_t q0 = (int64_t)seq * a.qs[0] + t * a.qs[1] + hq * a.qs[2];
            float f[NC][16], amax = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < 16; ++j) f[c][j] = 0.0f;
                if constexpr (HALVES) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (64 * c + 32 * e + 8 * g4 < a.D) load_values<DT, 8>(a.q, q0 + 64 * c + 32 * e + 8 * g4, a.qvec, f[c] + 8 * e);
                } else {
                    if (64 * c + 16 * g4 < a.D) load_values<DT, 16>(a.q, q0 + 64 * c + 16 * g4, a.qvec, f[c]);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(f[c][j]));
            }
            amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
            amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
            const int e = amax > 0.0f && isfinite(amax) ? ilogbf(amax) - 7 : 0;
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f;   // the largest product is then the largest score
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float x = ldexpf(sign * f[c][j], -e);
                    const _Float16 hi = (_Float16)x;
                    qf[n][0][c][j >> 3][j & 7] = hi;
                    if constexpr (TERMS == 2) qf[n][1][c][j >> 3][j & 7] = (_Float16)(x - (float)hi);
                }
            rs[n] = ldexpf(fabsf(a.scale) * kLog2e, e);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m[n] = w[n] = -INFINITY;
            l[n] = 0.0f;
        }
#pragma unroll
        for (int i = 32; i >= 1; i >>= 1) {
            largest = fmaxf(largest, __shfl_xor(largest, i, 64));
            const int x = __shfl_xor(whole, i, 64);
            whole = x < whole ? x : whole;
        }
        unit = __builtin_amdgcn_readfirstlane(largest > 0.0f ? ilogbf(largest) : 0);
        whole = __builtin_amdgcn_readfirstlane(whole);
    }

    // Block blk's products s with the queries, of scales ks and vs, to the weights pf of its values.
    __device__ __forceinline__ void weigh(f32x4 (&s)[NR][2], float ks, float vs, int blk, int lane, f16x8 (&pf)[NR][TERMS]) {
        const int g4 = lane >> 4;
        // log2 of the value scale is le + lm: where a later block, which some rows do not see, has values of the largest
        // size, vs 2^-unit may be too small for float32, and the sum of both parts has lost digits
        const float le = (float)(__builtin_amdgcn_frexp_expf(vs) - unit);
        float c[NR], lm[NR];   // c takes the products to units of log2
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            c[n] = rs[n] * ks;
            c[n] = c[n] == 0.0f ? 1e-30f : c[n];   // so that it leaves -inf what it is
            lm[n] = __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(vs));
        }
        if ((blk + 1) * kKvBlock > whole) {
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                if (blk * kKvBlock > last[n]) { c[n] = 1.0f; lm[n] = 0.0f; }   // a row that sees none of it, whatever its scales
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (blk * kKvBlock + 8 * g4 + j > last[n]) s[n][j >> 2][j & 3] = -INFINITY;
            }
        }
        float top[NR];
        bool passed = false;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            top[n] = s[n][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top[n] = fmaxf(top[n], s[n][j >> 2][j & 3]);
            top[n] *= c[n];
            passed = passed || top[n] > m[n] + kSlack || top[n] + (le + lm[n]) > w[n] + kSlack;
        }
        if (__any(passed)) {
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                float mx = fmaxf(top[n], __shfl_xor(top[n], 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = fmaxf(m[n], mx), wn = fmaxf(w[n], mx + (le + lm[n]));
                l[n] *= __builtin_amdgcn_exp2f(m[n] - (mn == -INFINITY ? 0.0f : mn));
                const float alpha = __builtin_amdgcn_exp2f(w[n] - (wn == -INFINITY ? 0.0f : wn));
                m[n] = mn;
                w[n] = wn;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[n][d] *= alpha;
            }
        }
        // exponentials with the value scale in them; l's are the same ones but for a factor, where that is not too far off
        bool far = false, large = TERMS == 2;
        float back[NR], from[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            from[n] = m[n] == -INFINITY ? 0.0f : m[n];
            back[n] = (le - ((w[n] == -INFINITY ? 0.0f : w[n]) - from[n])) + lm[n];
            far = far || !(fabsf(back[n]) < 60.0f);
            large = large || !(fabsf(from[n]) < kLarge);
        }
        if (TERMS == 2 || __any(large)) {   // the products become their distances from the maximum
#pragma unroll
            for (int n = 0; n < NR; ++n) {
#pragma unroll
                for (int j = 0; j < 8; ++j) s[n][j >> 2][j & 3] = __builtin_fmaf(s[n][j >> 2][j & 3], c[n], -from[n]);
                c[n] = 1.0f;
                from[n] = 0.0f;
            }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float add = back[n] + kWeightLog2, all = add - from[n];
            float sum = 0.0f, y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j >> 2][j & 3], c[n], all));
                sum += y[j];
                pf[n][0][j] = (_Float16)y[j];
                if constexpr (TERMS == 2) pf[n][1][j] = (_Float16)(y[j] - (float)pf[n][0][j]);
            }
            back[n] = __builtin_amdgcn_exp2f(-add) * sum;
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__any(far)) {
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                back[n] = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) back[n] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j >> 2][j & 3], c[n], -from[n]));
            }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) l[n] += back[n];
    }

    // l of whole rows.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            l[n] += __shfl_xor(l[n], 16, 64);
            l[n] += __shfl_xor(l[n], 32, 64);
        }
    }

    // The sums of piece n from w to count from ref, in one step: a power of two, and 2^-kSumLog2, which keeps sums of the
    // largest values finite, with it (w is -inf where a row saw nothing or values of 0).
    __device__ __forceinline__ void rescale(int n, float ref) {
        const float by = w[n] == -INFINITY ? 0.0f : w[n] - (ref == -INFINITY ? 0.0f : ref), whole_by = floorf(by);
        const float f = __builtin_amdgcn_exp2f(by - whole_by);
        const int e = (int)whole_by + unit - kWeightLog2 - kSumLog2;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][d][i] = ldexpf(o[n][d][i] * f, e);
    }

    __device__ __forceinline__ void store(const SharedArgs& a, int n, int r0, int64_t row0, float mt, float lt, int lane) const {
        const int r = r0 + 16 * n + (lane & 15), g4 = lane >> 4;
        if (r >= a.rows[S]) return;
        const int64_t at = row0 + r;
        if (g4 == 0) *reinterpret_cast<float2*>(a.stat[S] + 2 * at) = make_float2(mt, lt);
#pragma unroll
        for (int d = 0; d < ND; ++d)
            if (16 * d < a.D) *reinterpret_cast<f32x4*>(a.part[S] + at * a.D + 16 * d + 4 * g4) = o[n][d];
    }
};

// Up to 16 NR rows of one key head against blocks [b0, b1) of sequence `set` of a cache: S 0, a
// prefix (rows of all its W sequences), or 1, a sequence's own.
// SLOTS: of the wave's ring, 2 (the block that it computes on and the next one on its way) or 1.
template <int DT, int ND, int NR, int S, int SLOTS>
__device__ __forceinline__ void attend(const SharedArgs& a, char* ring, int set, int h, int rt, int b0, int b1,
                                       int64_t row0) {
    using R = Rows<DT, ND, NR, S>;
    constexpr int TERMS = R::TERMS, NC = R::NC;
    constexpr int kRing = SLOTS * kSlotBytes<ND>;
    static_assert(2 * NR * ND * 4 * 256 <= kSharedWaves * kRing, "the waves' sums fit the rings");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int len = clamp_length(a.lengths[S][set], a.nb[S]);
    const int64_t cell0 = ((int64_t)set * a.H + h) * a.nb[S];
    const int r0 = rt * NR * 16;
    char* my_ring = ring + wave * kRing;
    // the scales of the wave's next 64 blocks, one a lane; then the first blocks
    float ks64, vs64;
    auto load_scales = [&](int blk) {
        const int mine = blk + lane * kSharedWaves;
        ks64 = mine < b1 ? a.ks[S][cell0 + mine] : 0.0f;
        vs64 = mine < b1 ? a.vs[S][cell0 + mine] : 0.0f;
    };
    load_scales(b0 + wave);
    if (b0 + wave < b1) fetch_block<ND>(my_ring, a.kc[S], a.vc[S], cell0 + b0 + wave, a.D, lane);
    R rows;
    float largest = 0.0f;
    for (int i = b0 + lane; i < b1; i += 64) largest = fmaxf(largest, a.vs[S][cell0 + i]);
    rows.template init<false>(a, set, h, r0, len, largest, lane);
    // fragments: key row 8 (n16 / 4) + 4 tt + n16 % 4, piece 4 c + g4; value row 16 d + n16, keys 8 g4 .. 8 g4 + 7
    const int key_row = 8 * (n16 >> 2) + (n16 & 3);
    const int key_at = (key_row * kRow<ND> + (g4 ^ key_turn<ND>(key_row))) * 16;
    const int value_at = kKeyBytes<ND> + (n16 * 2 + ((g4 >> 1) ^ (n16 >> 3))) * 16 + (g4 & 1) * 8;
    asm volatile("" : "+v"(ks64), "+v"(vs64));   // they are here
    int step = 0, at = 0;   // the slot of the block
    for (int blk = b0 + wave; blk < b1; blk += kSharedWaves, ++step) {
        // the block is there
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
        asm volatile("" ::: "memory");
        if (step % 64 == 0 && step) {
            load_scales(blk);
            asm volatile("" : "+v"(ks64), "+v"(vs64));
        }
        const float ks = lane_value(ks64, step % 64), vs = lane_value(vs64, step % 64);
        const char* slot = my_ring + at * kSlotBytes<ND>;
        // the slot of the block before is free: all reads of it have come back, for its products are done
        if constexpr (SLOTS == 2) {
            at ^= 1;
            if (blk + kSharedWaves < b1) fetch_block<ND>(my_ring + at * kSlotBytes<ND>, a.kc[S], a.vc[S], cell0 + blk + kSharedWaves, a.D, lane);
        }
        // Codes are read a step ahead, and the steps stand apart (sched_barrier): else the compiler, with all reads
        // first, wants more registers than there are.
        f32x4 s[NR][2];
        auto key_codes = [&](int i) {
            return *reinterpret_cast<const u32x4*>(slot + (key_at ^ i / 2 * 64) + i % 2 * 4 * kRow<ND> * 16);
        };
        auto value_codes = [&](int d) { return *reinterpret_cast<const uint2*>(slot + value_at + d * 512); };
#pragma unroll
        for (int n = 0; n < NR; ++n) s[n][0] = s[n][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        u32x4 k = key_codes(0);
#pragma unroll
        for (int i = 0; i < 2 * NC; ++i) {   // both 16-key halves in turn: products that do not wait for each other
            const u32x4 next_k = key_codes(i + 1 < 2 * NC ? i + 1 : i);
            const f16x8 k0 = codes_f16<false>(k.x, k.y), k1 = codes_f16<false>(k.z, k.w);
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int u = 0; u < TERMS; ++u) s[n][i % 2] = mma(k0, rows.qf[n][u][i / 2][0], s[n][i % 2]);
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int u = 0; u < TERMS; ++u) s[n][i % 2] = mma(k1, rows.qf[n][u][i / 2][1], s[n][i % 2]);
            k = next_k;
            __builtin_amdgcn_sched_barrier(0);
        }
        uint2 v = value_codes(0);
        f16x8 pf[NR][TERMS];
        rows.weigh(s, ks, vs, blk, lane, pf);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const uint2 next_v = value_codes(d + 1 < ND ? d + 1 : d);
            const f16x8 vf = codes_f16<false>(v.x, v.y);
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int u = 0; u < TERMS; ++u) rows.o[n][d] = mma(vf, pf[n][u], rows.o[n][d]);
            v = next_v;
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (SLOTS == 1) {
            asm volatile("" ::: "memory");
            if (blk + kSharedWaves < b1) fetch_block<ND>(my_ring, a.kc[S], a.vc[S], cell0 + blk + kSharedWaves, a.D, lane);
        }
    }
    // join the waves: the four lanes of a row, then the upper half of the waves into the lower
    auto stats_of = [&](int i) { return reinterpret_cast<float2*>(ring + i * kRing); };
    rows.finish();
#pragma unroll
    for (int n = 0; n < NR; ++n)
        if (g4 == 0) stats_of(wave)[16 * n + n16] = make_float2(rows.m[n], rows.l[n]);
    __syncthreads();
    auto* sums = reinterpret_cast<float(*)[NR * ND * 4][64]>(ring);
    float lt[NR], mt[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        float2 st[kSharedWaves];
        mt[n] = -INFINITY;
#pragma unroll
        for (int i = 0; i < kSharedWaves; ++i) {
            st[i] = stats_of(i)[16 * n + n16];
            mt[n] = fmaxf(mt[n], st[i].x);
        }
        lt[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSharedWaves; ++i)
            lt[n] += st[i].y * __builtin_amdgcn_exp2f(st[i].x - (mt[n] == -INFINITY ? 0.0f : mt[n]));
        rows.rescale(n, mt[n]);
    }
    __syncthreads();
#pragma unroll
    for (int half = kSharedWaves / 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int i = 0; i < NR * ND * 4; ++i) sums[wave - half][i][lane] = rows.o[i / (ND * 4)][i / 4 % ND][i % 4];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int i = 0; i < NR * ND * 4; ++i) rows.o[i / (ND * 4)][i / 4 % ND][i % 4] += sums[wave][i][lane];
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int n = 0; n < NR; ++n) rows.store(a, n, r0, row0, mt[n], lt[n], lane);
}

// The form for many rows of a prefix: each wave has 16 rows of its own, and all take each
// block.  Its codes are turned into f16 once for all of them, in registers on their way from memory to LDS: one buffer
// is computed on while the next block's goes into the other, a barrier a block.
// LDS: key rows of kWideRow 16-byte pieces, piece j of row 8 a + 4 tt + b in place j ^ turn; value rows of 32 keys, piece j of
// row d in place j ^ value_place: an instruction serves lanes 0 .. 3, 12 .. 15, 20 .. 27 at once, and the like.
template <int ND> constexpr int kWideRow = ND <= 4 ? 8 : 16;
template <int ND> constexpr int kWideKeys = kKvBlock * kWideRow<ND> * 16;
template <int ND> constexpr int kWideBytes = kWideKeys<ND> + ND * 1024;
template <int ND> __device__ __forceinline__ int wide_turn(int r) {
    return kWideRow<ND> == 8 ? ((r >> 3) & 3) << 1 | (r & 3) >> 1 : ((r >> 3) & 3) << 2 | (r & 3);
}

__device__ __forceinline__ int value_place(int d) { return -(d >> 2) & 3; }

// 16 codes of a thread: piece i of 4 D in a block's 2 D of keys and 2 D of values.
struct WideCodes {
    u32x4 c[2];
};
__device__ __forceinline__ void load_codes(WideCodes& x, const int8_t* kc, const int8_t* vc, int64_t cell, int D) {
    const int64_t base = cell * kKvBlock * D;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = threadIdx.x + e * kSharedThreads;
        if (i < 4 * D) x.c[e] = *reinterpret_cast<const u32x4*>((i < 2 * D ? kc : vc - 32 * D) + base + i * 16);
    }
}
template <int ND>
__device__ __forceinline__ void spread_codes(char* tile, const WideCodes& x, const int (&to)[2][2], int D) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if ((int)threadIdx.x + e * kSharedThreads >= 4 * D) continue;
        *reinterpret_cast<f16x8*>(tile + to[e][0]) = codes_f16<false>(x.c[e].x, x.c[e].y);
        *reinterpret_cast<f16x8*>(tile + to[e][1]) = codes_f16<false>(x.c[e].z, x.c[e].w);
    }
}

template <int DT, int ND>
__device__ __forceinline__ void attend_wide(const SharedArgs& a, char* lds, int set, int h, int rt, int b0, int b1, int64_t row0) {
    using R = Rows<DT, ND, 1, 0>;
    constexpr int TERMS = R::TERMS, NC = R::NC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int len = clamp_length(a.lengths[0][set], a.nb[0]);
    const int64_t cell0 = ((int64_t)set * a.H + h) * a.nb[0];
    const int r0 = (rt * kSharedWaves + wave) * 16;
    const bool rows_here = r0 < a.rows[0];   // the other waves only turn codes
    // where the thread's codes go: keys, row i / (D / 16), pieces 2 (i % (D / 16)) and the next; values, row i / 2, pieces
    // 2 (i % 2) and the next
    int to[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        int i = threadIdx.x + e * kSharedThreads;
        const bool value = i >= 2 * a.D;
        i -= value ? 2 * a.D : 0;
        const int per = value ? 2 : a.D / 16, row = i / per, j = 2 * (i % per);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            to[e][u] = value ? kWideKeys<ND> + row * 64 + ((j + u) ^ value_place(row)) * 16
                             : (row * kWideRow<ND> + ((j + u) ^ wide_turn<ND>(row))) * 16;
    }
    float ks64, vs64;
    auto load_scales = [&](int blk) {
        ks64 = blk + lane < b1 ? a.ks[0][cell0 + blk + lane] : 0.0f;
        vs64 = blk + lane < b1 ? a.vs[0][cell0 + blk + lane] : 0.0f;
    };
    load_scales(b0);
    WideCodes raw[2];
    if (b0 < b1) load_codes(raw[0], a.kc[0], a.vc[0], cell0 + b0, a.D);
    if (b0 + 1 < b1) load_codes(raw[1], a.kc[0], a.vc[0], cell0 + b0 + 1, a.D);
    // what no code goes to is read all the same (heads of 80): zeros
    if (16 * ND != a.D)
        for (int i = threadIdx.x; i < 2 * kWideBytes<ND> / 16; i += kSharedThreads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    R rows;
    float largest = 0.0f;
    for (int i = b0 + lane; i < b1; i += 64) largest = fmaxf(largest, a.vs[0][cell0 + i]);
    rows.template init<true>(a, set, h, r0, len, largest, lane);
    const int key_row = 8 * (n16 >> 2) + (n16 & 3);
    const int key_at = (key_row * kWideRow<ND> + (g4 ^ wide_turn<ND>(key_row))) * 16;
    const int value_at = kWideKeys<ND> + n16 * 64 + (g4 ^ value_place(n16)) * 16;
    __syncthreads();
    if (b0 < b1) spread_codes<ND>(lds, raw[0], to, a.D);
    if (b0 + 2 < b1) load_codes(raw[0], a.kc[0], a.vc[0], cell0 + b0 + 2, a.D);
    // raw[1] holds the next block; raw[0] the one after it, on its way
    auto body = [&](int blk, int step, const char* tile, char* other, WideCodes& next) {
        // every wave has written its part of the tile, and read the other one
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): loads from memory stay on their way
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (step % 64 == 0 && step) load_scales(blk);
        const float ks = lane_value(ks64, step % 64), vs = lane_value(vs64, step % 64);
        if (rows_here) {
            f32x4 s[1][2] = {};
            auto key_codes = [&](int i) {
                return *reinterpret_cast<const f16x8*>(tile + (key_at ^ i / 2 * 64) + i % 2 * 4 * kWideRow<ND> * 16);
            };
            auto value_codes = [&](int d) { return *reinterpret_cast<const f16x8*>(tile + value_at + d * 1024); };
#pragma unroll
            for (int i = 0; i < 4 * NC; ++i) {
                if (i / 2 * 2 >= ND) continue;   // past the head
                const f16x8 k = key_codes(i);
#pragma unroll
                for (int u = 0; u < TERMS; ++u) s[0][i % 2] = mma(k, rows.qf[0][u][i / 4][i / 2 % 2], s[0][i % 2]);
            }
            f16x8 pf[1][TERMS];
            rows.weigh(s, ks, vs, blk, lane, pf);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const f16x8 v = value_codes(d);
#pragma unroll
                for (int u = 0; u < TERMS; ++u) rows.o[0][d] = mma(v, pf[0][u], rows.o[0][d]);
            }
        }
        if (blk + 1 < b1) spread_codes<ND>(other, next, to, a.D);
        if (blk + 3 < b1) load_codes(next, a.kc[0], a.vc[0], cell0 + blk + 3, a.D);
    };
    for (int blk = b0, step = 0; blk < b1; blk += 2, step += 2) {
        body(blk, step, lds, lds + kWideBytes<ND>, raw[1]);
        if (blk + 1 < b1) body(blk + 1, step + 1, lds + kWideBytes<ND>, lds, raw[0]);
    }
    if (!rows_here) return;
    rows.finish();
    rows.rescale(0, rows.m[0]);
    rows.store(a, 0, r0, row0, rows.m[0], rows.l[0], lane);
}

// NO: 16-row pieces of a sequence's own rows.  A prefix's go 16 to a wave, all four waves' against each block.  Heads of
// more than 128 values take the form with a ring (their tiles of f16, 28 to 32 KB each, are not built), for 16 rows (float32,
// whose two terms want the registers) or 32 (64 sequences of 4 heads on 8000 tokens, 256 values, 52 us, 16 rows 54; 192 values
// 43 and 46; where 16 rows are all, 8 sequences on 16000, 34 and 28.5).
template <int DT, int ND, int NO>
struct SharedForm {
    static constexpr bool kWide = ND <= 8;
    static constexpr int kPrefix = kWide ? 4 : DT == AXS6_F32 ? 1 : 2;   // 16-row pieces of a workgroup's
    static constexpr int kSlots = kWide ? 1 : 2;
    static constexpr int kRings = kSharedWaves * kSlots * kSlotBytes<ND>, kTiles = 2 * kWideBytes<ND>;
    static constexpr int kLds = kWide && kTiles > kRings ? kTiles : kRings;
    // waves a SIMD: as many as the registers allow
    static constexpr int kOccupancy = !kWide ? 1 : DT == AXS6_F32 ? (NO == 2 ? 2 : 3) : NO == 2 ? 3 : 4;
};

template <int DT, int ND, int NO>
__global__ __launch_bounds__(kSharedThreads, (SharedForm<DT, ND, NO>::kOccupancy)) void kv_shared_kernel(SharedArgs a) {
    using F = SharedForm<DT, ND, NO>;
    // The kernel's only LDS variable: beside a second one the compiler waits for all loads into LDS before any read of it.
    __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
    const int lane = threadIdx.x & 63;
    if ((int)blockIdx.x < a.prefix_groups) {
        // consecutive workgroups go round the 8 XCDs: the row tiles of a piece stay on one, whose
        // L2 then has its codes
        const int i = blockIdx.x >> 3, unit = i / a.row_tiles[0] * 8 + (blockIdx.x & 7), rt = i % a.row_tiles[0];
        if (unit >= a.units) return;
        const int piece = unit / a.H, h = unit % a.H;
        int p, b0, b1;
        if (a.even) {
            const Pieces c = even_pieces(a, lane);
            const uint64_t mine = __ballot(piece >= c.first && piece < c.first + c.count);
            if (!mine) return;
            p = __builtin_ctzll(mine);
            b0 = (piece - __shfl(c.first, p, 64)) * c.size;
            const int blocks = __shfl(c.blocks, p, 64);
            b1 = b0 + c.size < blocks ? b0 + c.size : blocks;
        } else {
            const int each = a.pieces[0] / a.P;
            p = piece / each;
            const int blocks = blocks_of(clamp_length(a.lengths[0][p], a.nb[0])), size = (blocks + each - 1) / each;
            b0 = piece % each * size;
            b1 = b0 + size < blocks ? b0 + size : blocks;
        }
        p = __builtin_amdgcn_readfirstlane(p);
        b0 = __builtin_amdgcn_readfirstlane(b0);
        b1 = __builtin_amdgcn_readfirstlane(b1);
        if constexpr (F::kWide) attend_wide<DT, ND>(a, lds, p, h, rt, b0, b1, (int64_t)unit * a.rows[0]);
        else attend<DT, ND, F::kPrefix, 0, F::kSlots>(a, lds, p, h, rt, b0, b1, (int64_t)unit * a.rows[0]);
    } else {
        const int i = blockIdx.x - a.prefix_groups, piece = i % a.pieces[1], j = i / a.pieces[1];
        const int rt = j % a.row_tiles[1], bh = j / a.row_tiles[1], b = bh / a.H, h = bh % a.H;
        const int len = clamp_length(a.lengths[1][b], a.nb[1]), blocks = blocks_of(len);
        const int size = (blocks + a.pieces[1] - 1) / a.pieces[1], b0 = piece * size;
        attend<DT, ND, NO, 1, F::kSlots>(a, lds, b, h, rt, b0, b0 + size < blocks ? b0 + size : blocks,
                              ((int64_t)piece * a.P * a.W * a.H + bh) * a.rows[1]);
    }
}

constexpr int kJoinSize = 256;

// GROUPS groups of D / 4 threads a row, which take every GROUPS-th of its pieces.
template <int DT, bool MANY>
__global__ __launch_bounds__(kJoinSize) void kv_shared_join_kernel(SharedArgs a) {
    using E = Elem<DT>;
    __shared__ int first_of[kMaxEven], count_of[kMaxEven];
    __shared__ float sh_m[kJoinSize], sh_l[kJoinSize];
    __shared__ f32x4 sh_o[kJoinSize];
    const int t = threadIdx.x, lanes = a.D / 4, groups = MANY ? kJoinSize / lanes : 1;
    if (a.even) {
        if (t < 64) {
            const Pieces c = even_pieces(a, t);
            if (t < kMaxEven) { first_of[t] = c.first; count_of[t] = c.count; }
        }
        __syncthreads();
    }
    const int64_t rows = (int64_t)a.P * a.W * a.H * a.rows[1];
    const int64_t i = MANY ? (int64_t)t : (int64_t)blockIdx.x * kJoinSize + t;
    const int64_t row = MANY ? (int64_t)blockIdx.x : i / lanes;
    const int g = MANY ? t / lanes : 0, d = (int)(MANY ? t % lanes : i % lanes) * 4;
    const bool here = row < rows && g < groups;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    int64_t bh = 0;
    int r = 0;
    if (here) {
        bh = row / a.rows[1];
        r = (int)(row - bh * a.rows[1]);
        const int b = (int)(bh / a.H), h = (int)(bh % a.H), p = b / a.W;
        const int each = a.even ? 0 : a.pieces[0] / a.P;
        const int first = a.even ? first_of[p] : p * each, count = a.even ? count_of[p] : each;
        const int64_t of_prefix = (int64_t)h * a.rows[0] + (int64_t)(b - p * a.W) * a.rows[1] + r;
        const int pieces = count + a.pieces[1];
        auto add = [&](int s) {
            const int S = s < count ? 0 : 1;
            const int64_t at = S == 0 ? (int64_t)(first + s) * a.H * a.rows[0] + of_prefix
                                      : (s - count) * rows + row;
            const float2 st = *reinterpret_cast<const float2*>(a.stat[S] + 2 * at);
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.part[S] + at * a.D + d);
            const float mn = fmaxf(m, st.x), ref = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - ref), fx = __builtin_amdgcn_exp2f(st.x - ref);
            o = o * f + x * fx;
            l = l * f + st.y * fx;
            m = mn;
        };
#pragma unroll 4
        for (int s = g; s < pieces; s += groups) add(s);
    }
    if constexpr (MANY) {
        sh_m[t] = m;
        sh_l[t] = l;
        sh_o[t] = o;
        __syncthreads();
        if (!here || g != 0) return;
        float top = m;
        for (int j = 1; j < groups; ++j) top = fmaxf(top, sh_m[j * lanes + t]);
        const float ref = top == -INFINITY ? 0.0f : top, f = __builtin_amdgcn_exp2f(m - ref);
        o *= f;
        l *= f;
        for (int j = 1; j < groups; ++j) {
            const float fj = __builtin_amdgcn_exp2f(sh_m[j * lanes + t] - ref);
            o += sh_o[j * lanes + t] * fj;
            l += sh_l[j * lanes + t] * fj;
        }
    } else if (!here) {
        return;
    }
    const float rl = l == 0.0f ? 0.0f : kSumScale / l;
    const int64_t b = bh / a.H;
    const int q = r / a.G, hq = (int)(bh % a.H) * a.G + r % a.G;
    auto* out = reinterpret_cast<typename E::S*>(a.out) + ((b * a.Tq + q) * a.H * a.G + hq) * a.D + d;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = E::from_f(o[j] * rl);
}

constexpr int kFewest = 2;   // blocks of a piece (4 beams on 300 tokens: 2 12.6 us, 4 14.7, 8 15.8)

// How a call is laid out.
struct SharedPlan {
    int np, no, even;
    int64_t pieces[2], row_tiles[2];
};
SharedPlan shared_plan(int dtype, int64_t P, int64_t W, int64_t H, int64_t rows, int64_t D, int64_t prefix_blocks,
                       int64_t blocks) {
    SharedPlan p;
    p.np = D <= 128 ? 4 : dtype == AXS6_F32 ? 1 : 2;
    // (512 queries of 4 heads, bf16, 45 us, 16 rows a wave 48; float32, 40 rows, 76 and 54)
    p.no = D > 128 || rows <= 16 ? 1 : 2;
    p.row_tiles[0] = (W * rows + 16 * p.np - 1) / (16 * p.np);
    p.row_tiles[1] = (rows + 16 * p.no - 1) / (16 * p.no);
    // seven of eight workgroups that the card holds, of some blocks each (four of eight: one prefix of 65536 tokens 37.5 ->
    // 43.9 us, 32000 for 128 sequences 148 -> 156, 3 x 21 sequences of 5 queries 37.8 -> 35; all of them 8 x 8 sequences on
    // 16383 75 -> 79; twice as many: hardly a case as short)
    const int64_t most = 224 * (D > 128 ? 1 : dtype == AXS6_F32 ? (p.no == 2 ? 2 : 3) : p.no == 2 ? 3 : 4);
    const int64_t groups = H * p.row_tiles[0], some = P * ((prefix_blocks + kFewest - 1) / kFewest);
    int64_t n = (most + groups - 1) / groups;
    n = n < some ? n : some;
    p.even = P <= kMaxEven;
    p.pieces[0] = p.even ? n + P - 1 : P * ((n + P - 1) / P);
    const int64_t own = P * W * H * p.row_tiles[1];
    n = (most + own - 1) / own;
    p.pieces[1] = n < (blocks + kFewest - 1) / kFewest ? n : (blocks + kFewest - 1) / kFewest;
    return p;
}

template <int DT, int ND>
void launch_shared(const SharedArgs& a, const SharedPlan& p, unsigned grid, hipStream_t st) {
    if constexpr (ND <= 8)
        if (p.no == 2) {
            kv_shared_kernel<DT, ND, 2><<<grid, kSharedThreads, 0, st>>>(a);
            return;
        }
    kv_shared_kernel<DT, ND, 1><<<grid, kSharedThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int64_t axs6_kv_shared_attention_workspace(int32_t dtype, int64_t P, int64_t W, int64_t Tq, int64_t Hq, int64_t H,
                                                      int64_t D, int64_t prefix_blocks, int64_t blocks) {
    if (!valid_dtype(dtype) || P <= 0 || W <= 0 || Tq <= 0 || H <= 0 || Hq <= 0 || Hq % H || D <= 0 || prefix_blocks <= 0 ||
        blocks < 0)
        return 0;
    const int64_t rows = Tq * (Hq / H);
    const SharedPlan p = shared_plan(dtype, P, W, H, rows, D, prefix_blocks, blocks);
    return (p.pieces[0] + p.pieces[1] * P) * W * H * rows * (D + 2) * (int64_t)sizeof(float);
}

extern "C" int axs6_kv_shared_attention(const void* q, int32_t dtype, int64_t P, int64_t W, int64_t Tq, int64_t Hq,
                                        int64_t H, int64_t D, const int64_t* q_strides, const void* pk_codes,
                                        const float* pk_scales, const void* pv_codes, const float* pv_scales,
                                        int64_t prefix_blocks, const int64_t* prefix_lengths, const void* k_codes,
                                        const float* k_scales, const void* v_codes, const float* v_scales, int64_t blocks,
                                        const int64_t* lengths, float scale, void* out, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    const char* fn = "axs6_kv_shared_attention";
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    constexpr int64_t kMost = ((int64_t)1 << 31) - 1;
    if (P < 0 || W < 0 || P > kMost || W > kMost || P * W > kMost)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: bad number of sequences", fn);
    int rc = check_cache(fn, P, H, D, prefix_blocks, pk_codes, pk_scales, pv_codes, pv_scales);
    if (rc) return rc;
    const int64_t B = P * W;
    rc = check_cache(fn, B, H, D, blocks, k_codes, k_scales, v_codes, v_scales);
    if (rc) return rc;
    if (Tq < 0 || Hq < 0 || (H > 0 && Hq % H))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: %lld query heads for %lld key heads", fn, (long long)Hq, (long long)H);
    if (!isfinite(scale)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: the scale must be finite", fn);
    if (B * Tq * Hq == 0) return AXS6_OK;
    if (H == 0 || prefix_blocks == 0) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: an empty prefix", fn);
    if (!q || !q_strides || !prefix_lengths || !lengths || !out)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null operand", fn);
    const int64_t es = dtype == AXS6_F32 ? 4 : 2, vl = 16 / es, rows = Tq * (Hq / H);
    if (Tq > (1 << 24) || Hq / H > (1 << 24) || rows > (1 << 24) || W * rows > (1 << 24) || B * H * rows > kMost / 64)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    if ((uintptr_t)q % es || (uintptr_t)out % es)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not element-aligned", fn);
    const int64_t need = axs6_kv_shared_attention_workspace(dtype, P, W, Tq, Hq, H, D, prefix_blocks, blocks);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld bytes required, got %lld", fn,
                    (long long)need, (long long)workspace_bytes);
    const SharedPlan p = shared_plan(dtype, P, W, H, rows, D, prefix_blocks, blocks);
    SharedArgs a{};
    a.q = q; a.out = out; a.scale = scale;
    a.qvec = (uintptr_t)q % 16 == 0;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = q_strides[i];
        a.qvec = a.qvec && q_strides[i] % vl == 0;
    }
    a.kc[0] = reinterpret_cast<const int8_t*>(pk_codes); a.vc[0] = reinterpret_cast<const int8_t*>(pv_codes);
    a.ks[0] = pk_scales; a.vs[0] = pv_scales; a.lengths[0] = prefix_lengths; a.nb[0] = (int)prefix_blocks;
    a.kc[1] = reinterpret_cast<const int8_t*>(k_codes); a.vc[1] = reinterpret_cast<const int8_t*>(v_codes);
    a.ks[1] = k_scales; a.vs[1] = v_scales; a.lengths[1] = lengths; a.nb[1] = (int)blocks;
    a.P = (int)P; a.W = (int)W; a.H = (int)H; a.G = (int)(Hq / H); a.Tq = (int)Tq; a.D = (int)D;
    a.rows[0] = (int)(W * rows); a.rows[1] = (int)rows;
    for (int i = 0; i < 2; ++i) { a.row_tiles[i] = (int)p.row_tiles[i]; a.pieces[i] = (int)p.pieces[i]; }
    a.even = p.even;
    const int64_t units = p.pieces[0] * H, prefix_groups = (units + 7) / 8 * 8 * p.row_tiles[0];
    const int64_t grid = prefix_groups + B * H * p.row_tiles[1] * p.pieces[1];
    if (grid > kMost) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    a.units = (int)units;
    a.prefix_groups = (int)prefix_groups;
    const int64_t rows0 = (int64_t)p.pieces[0] * H * a.rows[0], rows1 = (int64_t)p.pieces[1] * B * H * rows;
    a.part[0] = reinterpret_cast<float*>(workspace);
    a.part[1] = a.part[0] + rows0 * D;
    a.stat[0] = a.part[1] + rows1 * D;
    a.stat[1] = a.stat[0] + rows0 * 2;
    hipStream_t st = (hipStream_t)stream;
    by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (D <= 64) launch_shared<DT, 4>(a, p, (unsigned)grid, st);
        else if (D <= 96) launch_shared<DT, 6>(a, p, (unsigned)grid, st);
        else if (D <= 128) launch_shared<DT, 8>(a, p, (unsigned)grid, st);
        else if (D <= 192) launch_shared<DT, 12>(a, p, (unsigned)grid, st);
        else launch_shared<DT, 16>(a, p, (unsigned)grid, st);
        const int64_t all = B * H * rows, lanes = D / 4;
        // a workgroup a row where there are few (one prefix of 65536 tokens, 32 rows: 37.5 us, else 52.8; 4096 rows 27.4, so
        // 33.1)
        if (all < 1024) kv_shared_join_kernel<DT, true><<<(unsigned)all, kJoinSize, 0, st>>>(a);
        else kv_shared_join_kernel<DT, false><<<(unsigned)((all * lanes + kJoinSize - 1) / kJoinSize), kJoinSize, 0, st>>>(a);
    });
    return check_launch(fn);
}
