// Beam search's selection: of each sequence's W beams and their V continuations the
// `count` best.
//
// Beam w of a sequence has the score c_w and the logits z_w[V]; a candidate is
//   s_wj = c_w + ((z_wj - m_w) - log sum_j exp(z_wj - m_w)),   m_w the largest logit,
// and a beam that has ended offers one, (end, c_w).  The largest come first, equal ones
// in the order of w V + j.  No candidate: z_wj = -inf, and all of a beam of score -inf.
// A NaN or +inf in a logit or score that counts makes the sequence's results NaN.
//
// Order between beams needs more than 32 bits (float32 sums of some 100000
// exponentials move a score by 1e-6, and of many candidates two always lie that near):
// exponentials are float32, their sums and everything after float64.
//
// Two launches.  The first reads the logits once, four 16-byte vectors a lane at a time, and leaves
// the sum of exponentials and the maximum of each segment.  The second, a
// workgroup a sequence, needs few logits again: the K best candidates lie in the K
// best segments (K segments with a larger maximum, or an equal one further ahead, hold
// K candidates that come before any of another segment), whose logits it reads, and of
// these few reach the last such segment's maximum.  Where many do (few segments, equal values) the same choice is made
// among those segments' 16-byte vectors first.
//
// Bound by HBM where there are many rows, else by the second launch's chain of short steps on one CU a sequence.  Measured
// (first + second launch): 64 x 8 rows of 128000 bf16, 16 chosen, 29 + 14 us, the first at 4.5 TB/s; 3 x 48 of 50001 f16,
// 48 chosen, 9 + 16; 8 x 8 of 32000 f32, 16 chosen, 5.4 + 12; 4 rows of 256 4.4 + 8.  Of the second's 15 us at 3 x 48:
// the rows' sums 2.8, reading and scoring 4704 segments 3.1, the cut to 160 of them 2.8, ranking 1, reading and scoring the
// chosen ones' 3072 vectors, three a thread, 4.2, ranking 1.  Eight loads ahead instead of four there, or scoring whole
// vectors of which one logit counts, took 1 to 5 us more.  (Eight exponentials added in float32 before the float64 sum:
// 64 x 8 rows 39.8 us in all for 41.3, and scores of rows with one likely token off by 2e-7.)
#include <math.h>

#include "axs6_internal.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

constexpr int kRowWaves = 4;
constexpr int kLoads = 4;        // vectors of a lane in a segment
constexpr int kSelThreads = 1024;
constexpr int kMaxBeams = AXS6_BEAM_MAX_BEAMS, kMaxCount = AXS6_BEAM_MAX_COUNT;
constexpr int kList = 256;       // items that are ranked by comparing all with all: at most these,
constexpr int kDirect = 160;     // and from here on a cut pays (the work grows with the square)
constexpr int kBins = 2048;
constexpr int kAhead = 4;        // vectors of the chosen segments that a thread has on their way
constexpr int kHeld = 8;         // items that a thread holds
static_assert(kMaxCount <= kDirect && kDirect <= kList);
constexpr float kLog2e = 1.4426950408889634f;
// log2(e) minus its float32
constexpr float kLog2eLow = 1.92596299e-8f;

struct BeamArgs {
    const void* logits;
    int64_t ld_seq, ld_beam;      // in elements
    const float* scores;
    const uint8_t* finished;
    int64_t end;
    int W, V, units, chunks, count;
    int segs, vecs_log2;          // segments of a row, and 16-byte vectors of one
    float* seg_max;               // (G * W, segs)
    double2* part;                // (G * W, chunks): maximum, sum of exponentials
    float* out_scores;
    int64_t *parents, *tokens;
};

// Whether beam `row` has logits that count.
__device__ __forceinline__ bool live(const BeamArgs& a, int64_t row) {
    return !(a.finished && a.finished[row]) && a.scores[row] != -INFINITY;
}

// A vector of a row's logits from element i; -inf past its end.  No alignment is needed.
template <int DT>
__device__ __forceinline__ u32x4 load_vector(const typename Elem<DT>::S* z, int64_t i, int64_t V) {
    using E = Elem<DT>;
    typedef u32x4 __attribute__((aligned(2))) loose;
    if (i + E::V <= V) return *reinterpret_cast<const loose*>(z + i);
    float x[E::V];
#pragma unroll
    for (int j = 0; j < E::V; ++j) x[j] = i + j < V ? E::to_f(z[i + j]) : -INFINITY;
    return E::pack(x);
}

template <int CTRL>
__device__ __forceinline__ float max_dpp(float v) {
    const int x = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
    return fmaxf(v, __builtin_bit_cast(float, x));
}
// Of 16 lanes; of all, from those.
__device__ __forceinline__ float max16(float v) {
    v = max_dpp<0xb1>(v);
    v = max_dpp<0x4e>(v);
    v = max_dpp<0x141>(v);
    return max_dpp<0x140>(v);
}
__device__ __forceinline__ float max64(float of16) {
    float r = -INFINITY;
#pragma unroll
    for (int i = 0; i < 64; i += 16)
        r = fmaxf(r, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, of16), i)));
    return r;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// exp(x - m): the constant's second half counts, for the same m stands in all of a row's terms
__device__ __forceinline__ float exp_diff(float x, float m) {
    const float d = x - m;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, kLog2e, d * kLog2eLow));
}

// Chunk blockIdx.x of row blockIdx.y: units of four vectors a lane, to its waves in turn.  LEVEL: a segment is 0 a vector
// of 16 lanes, 1 one of all, 2 all four.
template <int DT, int LEVEL>
__global__ __launch_bounds__(64 * kRowWaves) void beam_rows_kernel(BeamArgs a) {
    using E = Elem<DT>;
    constexpr int PART = 64 * E::V;
    __shared__ double sh_s[kRowWaves];
    __shared__ float sh_m[kRowWaves];
    const int64_t row = blockIdx.y;
    if (!live(a, row)) return;
    const auto* z = reinterpret_cast<const typename E::S*>(a.logits) + row / a.W * a.ld_seq + row % a.W * a.ld_beam;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = (a.units + a.chunks - 1) / a.chunks, s0 = blockIdx.x * per, s1 = s0 + per < a.units ? s0 + per : a.units;
    float m = -INFINITY;
    double sum = 0.0;
    u32x4 raw[kLoads], next[kLoads];
    auto load = [&](int s) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) next[i] = load_vector<DT>(z, ((int64_t)s * kLoads + i) * PART + lane * E::V, a.V);
    };
    if (s0 + w < s1) load(s0 + w);
    for (int s = s0 + w; s < s1; s += kRowWaves) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) raw[i] = next[i];
        if (s + kRowWaves < s1) load(s + kRowWaves);
        float x[kLoads][E::V], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            E::unpack(raw[i], x[i]);
            float v = x[i][0];
#pragma unroll
            for (int j = 1; j < E::V; ++j) v = fmaxf(v, x[i][j]);
            if constexpr (LEVEL == 2) {
                top = fmaxf(top, v);
            } else {
                v = max16(v);
                const int seg = LEVEL == 0 ? (s * kLoads + i) * 4 + (lane >> 4) : s * kLoads + i;
                const float all = max64(v);
                if (lane % (LEVEL == 0 ? 16 : 64) == 0 && seg < a.segs) a.seg_max[row * a.segs + seg] = LEVEL == 0 ? v : all;
                top = fmaxf(top, all);
            }
        }
        if constexpr (LEVEL == 2) {
            top = max64(max16(top));
            if (lane == 0) a.seg_max[row * a.segs + s] = top;
        }
        if (top > m) {
            if (m != -INFINITY) sum *= exp((double)m - (double)top);
            m = top;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            double part = 0.0;
#pragma unroll
            for (int j = 0; j < E::V; ++j) part += exp_diff(x[i][j], ref);
            sum += part;
        }
    }
    sum = wave_sum(sum);
    if (lane == 0) { sh_m[w] = m; sh_s[w] = sum; }
    __syncthreads();
    if (threadIdx.x != 0) return;
    float mt = sh_m[0];
    for (int i = 1; i < kRowWaves; ++i) mt = fmaxf(mt, sh_m[i]);
    double st = 0.0;
    for (int i = 0; i < kRowWaves; ++i) st += sh_m[i] == mt ? sh_s[i] : sh_s[i] * exp((double)sh_m[i] - (double)mt);
    a.part[row * a.chunks + blockIdx.x] = make_double2(mt, st);
}

// Doubles in an order-preserving whole number, and back.
__device__ __forceinline__ uint64_t key_of(double d) {
    const uint64_t u = __builtin_bit_cast(uint64_t, d + 0.0);   // -0 as 0
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t k) {
    return __builtin_bit_cast(double, k >> 63 ? k & 0x7fffffffffffffffull : ~k);
}

struct Scratch {
    uint64_t key[kList];      // items to be ranked
    int id[kList], rank[kList];
    uint64_t best_key[kMaxCount];   // the choice
    int best_id[kMaxCount];
    int bins[kBins];
    uint64_t hi, lo;
    int above, more, listed, chosen, wave[kSelThreads / 64];
};

// One workgroup a sequence.  It chooses by turns: segments, where need be vectors of theirs, candidates; each time the K
// items of largest key (equal keys by the smaller id) of any number, 8192 and those chosen so far at a time, by the one
// piece of code in the loop (a workgroup runs it a few times only: most of its time would go into fetching more code).
// The interval [lo, hi] of keys in which the K-th lies is cut into 2048 bins, again and again, until what lies at or
// above it fits the list; keys that are all equal are cut by their ids instead.
template <int DT>
__global__ __launch_bounds__(kSelThreads) void beam_select_kernel(BeamArgs a) {
    using E = Elem<DT>;
    __shared__ double score[kMaxBeams], log_sum[kMaxBeams];   // a beam that has ended: log_sum = NaN
    __shared__ float largest[kMaxBeams];
    __shared__ Scratch s;
    __shared__ int source[kMaxCount], bad;   // the segments chosen, then the vectors
    __shared__ unsigned long long top;       // the best candidate's key
    // of a chosen segment: its beam (below 0: one that has ended, from -1 on), first token, and what its logits have to reach
    __shared__ int seg_beam[kMaxCount], seg_token[kMaxCount];
    __shared__ float seg_low[kMaxCount];
    const int64_t g = blockIdx.x, row0 = g * a.W;
    const int lane = threadIdx.x & 63, t = threadIdx.x, K = a.count;
    const int wave0 = __builtin_amdgcn_readfirstlane(t & ~63);   // the wave's first thread
    if (t == 0) {
        bad = 0;
        top = 0;
    }
    __syncthreads();
    // the rows' sums, 16 lanes a row
    for (int w0 = 0; w0 + wave0 / 16 < a.W; w0 += kSelThreads / 16) {
        const int w = w0 + t / 16, l16 = t & 15;
        const float c = w < a.W ? a.scores[row0 + w] : -INFINITY;
        const bool here = w < a.W && live(a, row0 + w);
        float m = -INFINITY;
        for (int i = l16; here && i < a.chunks; i += 16) m = fmaxf(m, (float)a.part[(row0 + w) * a.chunks + i].x);
        m = max16(m);
        double sum = 0.0;
#pragma unroll 1
        for (int i = l16; here && i < a.chunks; i += 16) {
            const double2 p = a.part[(row0 + w) * a.chunks + i];
            sum += p.x == m ? p.y : p.y * exp(p.x - m);
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (l16 == 0 && w < a.W) {
            double l = NAN;
            if (here) {
                l = m == -INFINITY && sum == 0.0 ? 0.0 : log(sum);   // nothing but -inf: no candidates
                if (l != l) bad = 1;                                 // +inf among the logits: inf - inf
            }
            if (!(c < INFINITY)) bad = 1;
            score[w] = c;
            largest[w] = m;
            log_sum[w] = l;
            // the beam's best candidate, where it has one
            if (here ? m != -INFINITY : c != -INFINITY) atomicMax(&top, (unsigned long long)key_of(here ? c + ((double)m - m - l) : c));
        }
    }
    for (int i = t; i < kBins; i += kSelThreads) s.bins[i] = 0;
    __syncthreads();
    if (bad) {
        for (int r = t; r < K; r += kSelThreads) {
            a.out_scores[g * K + r] = NAN;
            a.parents[g * K + r] = a.tokens[g * K + r] = 0;
        }
        return;
    }
    const auto* z0 = reinterpret_cast<const typename E::S*>(a.logits) + g * a.ld_seq;
    const int vecs = 1 << a.vecs_log2, row_vecs = a.segs << a.vecs_log2;
    auto key = [&](int w, float z) { return key_of(score[w] + (((double)z - largest[w]) - log_sum[w])); };
    auto ended = [&](int w) { return log_sum[w] != log_sum[w]; };
    uint64_t least = 0;   // what a candidate's key has to reach
    // vector v of the chosen segments
    auto read = [&](int v, int n) {
        u32x4 raw = {0, 0, 0, 0};
        if (v >= n) return raw;
        const int sg = v >> a.vecs_log2, w = seg_beam[sg], j = seg_token[sg] + (v & (vecs - 1)) * E::V;
        return w >= 0 && j < a.V ? load_vector<DT>(z0 + w * a.ld_beam, j, a.V) : raw;
    };
    // a bit for each of its values that may be a candidate; of an ended beam's first vector one
    auto reach = [&](int v, int n, u32x4 raw) {
        if (v >= n) return 0u;
        const int sg = v >> a.vecs_log2, w = seg_beam[sg], at = (v & (vecs - 1)) * E::V;
        const float low = seg_low[sg];
        float x[E::V];
        E::unpack(raw, x);
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < E::V; ++e) bits |= (uint32_t)(x[e] >= low && x[e] != -INFINITY) << e;
        return w < 0 ? (uint32_t)(at == 0) : seg_token[sg] + at < a.V ? bits : 0u;
    };
    // value e of it, where it is one
    auto candidate = [&](int v, int e, u32x4 raw, auto f) {
        const int sg = v >> a.vecs_log2, w = seg_beam[sg], j = seg_token[sg] + (v & (vecs - 1)) * E::V;
        float x[E::V];
        E::unpack(raw, x);
        float z = x[0];
#pragma unroll
        for (int i = 1; i < E::V; ++i) z = e == i ? x[i] : z;
        const uint64_t k = w < 0 ? key_of(score[-1 - w]) : key(w, z);
        if (k >= least) f(k, w < 0 ? (-1 - w) * a.V + (int)a.end : w * a.V + j + e);
    };
    auto list = [&](uint64_t k, int id) {
        const int at = atomicAdd(&s.listed, 1);
        if (at < kList) { s.key[at] = k; s.id[at] = id; }
    };
    enum { kSegments, kVectors, kTokens };
    int turn = kSegments, n = a.W * a.segs, done = 0, chosen = 0;   // items of the turn; those looked at; sources
    bool listed = false;   // what there is stands in the list already
    for (;;) {
        if (!listed) {
            // up to 8 items a thread, and the best of those before
            uint64_t held[kHeld + 1];
            int id[kHeld + 1];
            uint32_t some = 0;
            if (turn == kSegments) {   // of an ended beam its first stands for the end
                float z[kHeld];
#pragma unroll
                for (int q = 0; q < kHeld; ++q) {
                    const int i = done + q * kSelThreads + t;
                    z[q] = i < n ? a.seg_max[row0 * a.segs + i] : -INFINITY;
                }
#pragma unroll
                for (int q = 0; q < kHeld; ++q) {
                    held[q] = 0;
                    id[q] = 0;
                    if (done + q * kSelThreads + wave0 >= n) continue;
                    const int i = done + q * kSelThreads + t, w = (i < n ? i : 0) / a.segs;
                    const bool end = ended(w);
                    held[q] = end ? key_of(score[w]) : key(w, z[q]);
                    id[q] = i;
                    const bool is = i < n && score[w] != -INFINITY && (end ? i == w * a.segs : z[q] != -INFINITY);
                    some |= (uint32_t)is << q;
                }
            } else {
#pragma unroll
                for (int q = 0; q < kHeld; ++q) { held[q] = 0; id[q] = 0; }
#pragma unroll 1
                for (int q = 0; q < kHeld && done + q * kSelThreads + wave0 < n; ++q) {
                    const int i = done + q * kSelThreads + t;
                    uint64_t k = 0;
                    int d = 0;
                    bool is = false;
                    if (i < n && turn == kVectors) {
                        const u32x4 raw = read(i, n);
#pragma unroll 1
                        for (uint32_t hits = reach(i, n, raw); hits; hits &= hits - 1)
                            candidate(i, __builtin_ctz(hits), raw, [&](uint64_t x, int) { k = x > k ? x : k; });
                        d = (source[i >> a.vecs_log2] << a.vecs_log2) + (i & (vecs - 1));
                        is = k != 0;
                    } else if (i < n) {
                        const int v = source[i / E::V], w = v / row_vecs, j = (v - w * row_vecs) * E::V + i % E::V;
                        if (ended(w)) {
                            k = key_of(score[w]);
                            d = w * a.V + (int)a.end;
                            is = i % E::V == 0;
                        } else if (j < a.V) {
                            const float z = E::to_f(z0[w * a.ld_beam + j]);
                            k = key(w, z);
                            d = w * a.V + j;
                            is = z != -INFINITY && k >= least;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < kHeld; ++x)
                        if (x == q) { held[x] = k; id[x] = d; }
                    some |= (uint32_t)is << q;
                }
            }
            if (done && t < s.chosen) {
                held[kHeld] = s.best_key[t];
                id[kHeld] = s.best_id[t];
                some |= 1u << kHeld;
            }
            // Keys are first looked for within four powers of two of the largest that there is.
            if (t == 0) {
                s.hi = top;
                s.lo = n > kDirect && top > 1ull << 54 ? top - (1ull << 54) + 1 : 0;
                s.above = s.listed = 0;
                s.more = n > kDirect;
            }
            __syncthreads();
            bool by_id = false;
            uint64_t tied = 0;
            // (7 cuts of 11 bits end the keys, 3 the ids)
#pragma unroll 1
            for (int cut = 0; cut < 14 && s.more; ++cut) {
                const uint64_t H = s.hi, L = s.lo;
                const int above = s.above;
                const int bits = 64 - __builtin_clzll((H - L) | 1), shift = bits > 11 ? bits - 11 : 0;   // (H - L) >> shift < 2048
#pragma unroll
                for (int q = 0; q <= kHeld; ++q) {
                    uint64_t k = held[q];
                    const bool in = (some >> q & 1) && !(by_id && k != tied);
                    if (by_id) k = 0xffffffffull - (uint32_t)id[q];   // the smaller id first
                    if (in && k >= L && k <= H) atomicAdd(&s.bins[(H - k) >> shift], 1);
                }
                __syncthreads();
                // the bin in which the count passes K: each thread two bins, summed over waves
                const int c0 = s.bins[2 * t], c1 = s.bins[2 * t + 1];
                s.bins[2 * t] = s.bins[2 * t + 1] = 0;
                int before = c0 + c1;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int x = __shfl_up(before, o, 64);
                    if (lane >= o) before += x;
                }
                if (lane == 63) s.wave[t >> 6] = before;
                __syncthreads();
                int total = 0;
#pragma unroll
                for (int i = 0; i < kSelThreads / 64; ++i) {
                    const int x = s.wave[i];
                    before += i < (t >> 6) ? x : 0;
                    total += x;
                }
                before += above - c0 - c1;   // items of bins before this thread's, and above all
                int bin = -1, first = 0, in = 0;
                if (before < K && before + c0 >= K) { bin = 2 * t; first = before; in = c0; }
                else if (before + c0 < K && before + c0 + c1 >= K) { bin = 2 * t + 1; first = before + c0; in = c1; }
                if (above + total < K) {   // the K-th lies below the interval, or there is none
                    if (t == 0) {
                        s.more = L > 0 && !by_id;
                        s.hi = s.more ? L - 1 : H;
                        s.lo = 0;
                        s.above = above + total;
                    }
                } else if (bin >= 0) {
                    const uint64_t nh = H - ((uint64_t)bin << shift), width = ((uint64_t)1 << shift) - 1;
                    s.hi = nh;
                    s.lo = nh - L > width ? nh - width : L;
                    s.above = first;
                    s.more = first + in > kDirect;
                }
                __syncthreads();
                if (s.more && s.hi == s.lo && !by_id) {   // all equal, but for their ids, which are distinct
                    by_id = true;
                    tied = s.hi;
                    __syncthreads();
                    if (t == 0) { s.hi = 0xffffffffull; s.lo = 0; }
                    __syncthreads();
                }
            }
            const uint64_t L = s.lo;
#pragma unroll
            for (int q = 0; q <= kHeld; ++q) {
                if (!(some >> q & 1)) continue;
                const uint64_t k = held[q];
                if (by_id ? k > tied || (k == tied && 0xffffffffull - (uint32_t)id[q] >= L) : k >= L) list(k, id[q]);
            }
            done += kHeld * kSelThreads;
        } else {
            done = n;
        }
        // the list's K first: an item's place is the number of those before it, counted by several threads
        __syncthreads();
        const int m = s.listed < kList ? s.listed : kList;
        if (t < kList) s.rank[t] = 0;
        __syncthreads();
        int wide = 64;
        while (wide < m) wide *= 2;
        const int mine = t & (wide - 1), share = kSelThreads / wide;
        if (mine < m) {
            const uint64_t k = s.key[mine];
            const int d = s.id[mine];
            int before = 0;
#pragma unroll 4
            for (int x = t / wide; x < m; x += share) before += s.key[x] > k || (s.key[x] == k && s.id[x] < d);
            if (before) atomicAdd(&s.rank[mine], before);
        }
        __syncthreads();
        if (t < m && s.rank[t] < K) { s.best_key[s.rank[t]] = s.key[t]; s.best_id[s.rank[t]] = s.id[t]; }
        if (t == 0) s.chosen = m < K ? m : K;
        __syncthreads();
        if (done < n) continue;
        if (turn == kTokens || listed) break;
        // the chosen ones' candidates are none worse than the last one's best, where there are enough
        chosen = s.chosen;
        if (chosen == K && s.best_key[K - 1] > least) least = s.best_key[K - 1];
        if (t < chosen) {
            const int id = s.best_id[t];
            source[t] = id;
            if (turn == kSegments) {
                const int w = id / a.segs;
                seg_beam[t] = ended(w) ? -1 - w : w;
                seg_token[t] = ((id - w * a.segs) << a.vecs_log2) * E::V;
                // a logit below this is none of the candidates, by more than the rounding of either
                const double from = value_of(least), m = largest[w], l = log_sum[w];
                seg_low[t] = least ? (float)(from - score[w] + l + m - 1e-6 * (fabs(from) + fabs(score[w]) + l + fabs(m))) : -INFINITY;
            }
        }
        if (t == 0) s.listed = 0;
        __syncthreads();
        done = 0;
        if (turn == kVectors) {
            turn = kTokens;
            n = chosen * E::V;
            continue;
        }
        n = chosen << a.vecs_log2;
#pragma unroll 1
        for (int v = t; v - lane < n; v += kAhead * kSelThreads) {
            u32x4 raw[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) raw[i] = read(v + i * kSelThreads, n);
            // a bit for each value that may be a candidate: few have one, and the wave goes round as often as the lane with the most
            uint64_t hits = 0;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) hits |= (uint64_t)reach(v + i * kSelThreads, n, raw[i]) << (i * E::V);
#pragma unroll 1
            for (; hits; hits &= hits - 1) {
                const int at = __builtin_ctzll(hits), i = at / E::V;
                u32x4 r = raw[0];
#pragma unroll
                for (int q = 1; q < kAhead; ++q) r = i == q ? raw[q] : r;
                candidate(v + i * kSelThreads, at % E::V, r, list);
            }
        }
        __syncthreads();
        listed = s.listed <= kList;
        __syncthreads();   // all have read it: the next turn starts the list anew
        turn = kVectors;
    }
    for (int r = t; r < K; r += kSelThreads) {
        const bool some = r < s.chosen;
        a.out_scores[g * K + r] = some ? (float)value_of(s.best_key[r]) : -INFINITY;
        a.parents[g * K + r] = some ? s.best_id[r] / a.V : 0;
        a.tokens[g * K + r] = some ? s.best_id[r] % a.V : 0;
    }
}

// How a call is laid out: units of a row, workgroups that share one, and segments.
struct BeamPlan {
    int64_t units, chunks, segs;
    int level, vecs_log2;
};
BeamPlan beam_plan(int64_t rows, int64_t W, int64_t V, int64_t count, int dtype) {
    BeamPlan p;
    const int64_t vec = dtype == AXS6_F32 ? 4 : 8, unit = 64 * kLoads * vec;
    p.units = (V + unit - 1) / unit;
    // eight units a wave, or fewer where that makes less than 2048 workgroups (512: 3 x 48 rows of 50001 24.3 -> 26.0 us;
    // 8192: 64 x 8 of 128000 41.3 -> 44.2)
    int64_t per = 8 * kRowWaves;
    while (per > kRowWaves && rows * ((p.units + per - 1) / per) < 2048) per /= 2;
    p.chunks = (p.units + per - 1) / per;
    // The choice looks at all segments, 8192 at a time, and at the vectors of those chosen; up to 160 segments spare it
    // their cut.  Finer segments where that saves a quarter of this work (3 x 48 rows of 50001, an eighth), since
    // they cost the first launch some (64 x 8 of 128000 28.8 -> 31.3), and where there are not four times as many as
    // are chosen: with as many, the last one's maximum is low and most logits pass it.
    // In vectors' worth of time each further 8192 segments are 4096 (16384: 4 x 200 rows of 32000, 128 chosen, 57 -> 61 us;
    // 0: the same there, 1 x 64 of 128000 47 -> 41), the cut 2048 (0: 64 x 8 of 128000 41 -> 44, 2 x 2 of 300000 29 -> 27;
    // 8192: 64 x 64 of 1000 25 -> 27).
    int64_t least = -1;
    for (int level = 2; level >= 0; --level) {
        const int log2 = level == 2 ? 8 : level == 1 ? 6 : 4;
        const int64_t size = vec << log2, segs = (V + size - 1) / size, n = W * segs;
        const int64_t work = n + (n - 1) / (kHeld * kSelThreads) * 4096 + (n > kDirect ? 2048 : 0) + (count << log2);
        const bool few = n < 4 * count;
        if (least >= 0 && work > least / 4 * 3) break;
        p.level = level;
        p.vecs_log2 = log2;
        p.segs = segs;
        least = few ? INT64_MAX : work;
    }
    return p;
}

template <int DT>
void launch_beams(const BeamArgs& a, const BeamPlan& p, int64_t G, hipStream_t st) {
    const dim3 grid((unsigned)a.chunks, (unsigned)(G * a.W));
    if (p.level == 0) beam_rows_kernel<DT, 0><<<grid, 64 * kRowWaves, 0, st>>>(a);
    else if (p.level == 1) beam_rows_kernel<DT, 1><<<grid, 64 * kRowWaves, 0, st>>>(a);
    else beam_rows_kernel<DT, 2><<<grid, 64 * kRowWaves, 0, st>>>(a);
    beam_select_kernel<DT><<<(unsigned)G, kSelThreads, 0, st>>>(a);
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int64_t axs6_beam_select_workspace(int64_t G, int64_t W, int64_t V, int64_t count, int32_t dtype) {
    if (G <= 0 || W <= 0 || V <= 0 || count <= 0 || !valid_dtype(dtype)) return 0;
    const BeamPlan p = beam_plan(G * W, W, V, count, dtype);
    return G * W * p.chunks * (int64_t)sizeof(double2) + (G * W * p.segs + 3) / 4 * 16;
}

extern "C" int axs6_beam_select(const void* logits, int32_t dtype, int64_t G, int64_t W, int64_t V, int64_t ld_sequence,
                                int64_t ld_beam, const float* scores, const uint8_t* finished, int64_t end, int64_t count,
                                float* out_scores, int64_t* parents, int64_t* tokens, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    const char* fn = "axs6_beam_select";
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    if (G < 0 || W < 1 || V < 1) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: bad dimension", fn);
    if (count < 1 || count > kMaxCount || W > kMaxBeams)
        return fail(AXS6_ERR_UNSUPPORTED, "%s: 1 to %d candidates of up to %d beams, got %lld of %lld", fn, kMaxCount,
                    kMaxBeams, (long long)count, (long long)W);
    if (V > ((int64_t)1 << 31) - 1 || W * V > ((int64_t)1 << 31) - 1 || G * W > ((int64_t)1 << 31) - 1)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    if (G * W > 65535) return fail(AXS6_ERR_UNSUPPORTED, "%s: at most 65535 beams a call", fn);
    if (finished && (end < 0 || end >= V)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: end outside the vocabulary", fn);
    if (G == 0) return AXS6_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null operand", fn);
    if ((uintptr_t)logits % (dtype == AXS6_F32 ? 4 : 2))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not element-aligned", fn);
    const int64_t need = axs6_beam_select_workspace(G, W, V, count, dtype);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld bytes required, got %lld", fn,
                    (long long)need, (long long)workspace_bytes);
    BeamArgs a{};
    a.logits = logits; a.ld_seq = ld_sequence; a.ld_beam = ld_beam; a.scores = scores; a.finished = finished; a.end = end;
    a.W = (int)W; a.V = (int)V; a.count = (int)count;
    const BeamPlan p = beam_plan(G * W, W, V, count, dtype);
    a.units = (int)p.units; a.chunks = (int)p.chunks; a.segs = (int)p.segs; a.vecs_log2 = p.vecs_log2;
    a.part = reinterpret_cast<double2*>(workspace);
    a.seg_max = reinterpret_cast<float*>(a.part + G * W * a.chunks);
    a.out_scores = out_scores; a.parents = parents; a.tokens = tokens;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AXS6_F32) launch_beams<AXS6_F32>(a, p, G, st);
    else if (dtype == AXS6_BF16) launch_beams<AXS6_BF16>(a, p, G, st);
    else launch_beams<AXS6_F16>(a, p, G, st);
    return check_launch(fn);
}
