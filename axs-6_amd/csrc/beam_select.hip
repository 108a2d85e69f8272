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
// Two launches.  The first reads the logits once: a wave takes segments of 64 16-byte
// vectors and leaves each one's maximum and the sum of exponentials.  The second, a
// workgroup a sequence, needs few logits again: the K best candidates lie in the K
// best segments (K segments with a larger maximum, or an equal one further ahead, hold
// K candidates that come before any of another segment), whose logits it reads.  Both
// choices are one routine: the K first of n distinct keys (score, place).
// Bound by HBM: the logits, read once.
#include <math.h>

#include "axs6_internal.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

constexpr int kRowWaves = 4;
constexpr int kSelThreads = 1024;
constexpr int kMaxBeams = AXS6_BEAM_MAX_BEAMS, kMaxCount = AXS6_BEAM_MAX_COUNT;
constexpr int kList = 256;       // candidates that are ranked by comparing all with all; at least kMaxCount
constexpr int kBins = 2048;
constexpr float kLog2e = 1.4426950408889634f;
// log2(e) minus its float32
constexpr float kLog2eLow = 1.92596299e-8f;

struct BeamArgs {
    const void* logits;
    int64_t ld_seq, ld_beam;      // in elements
    const float* scores;
    const uint8_t* finished;
    int64_t end;
    int W, V, segs, chunks, count;
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
__device__ __forceinline__ void load_logits(const typename Elem<DT>::S* z, int64_t i, int64_t V, float* x) {
    using E = Elem<DT>;
    typedef u32x4 __attribute__((aligned(2))) loose;
    if (i + E::V <= V) {
        E::unpack(*reinterpret_cast<const loose*>(z + i), x);
    } else {
#pragma unroll
        for (int j = 0; j < E::V; ++j) x[j] = i + j < V ? E::to_f(z[i + j]) : -INFINITY;
    }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// x - m times log2(e): the constant's second half counts, for the same m stands in all of a row's terms
__device__ __forceinline__ float exp_diff(float x, float m) {
    const float d = x - m;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, kLog2e, d * kLog2eLow));
}

// Chunk blockIdx.x of row blockIdx.y: segments of 64 vectors, to its waves in turn.
template <int DT>
__global__ __launch_bounds__(64 * kRowWaves) void beam_rows_kernel(BeamArgs a) {
    using E = Elem<DT>;
    constexpr int SEG = 64 * E::V;
    __shared__ double sh_s[kRowWaves];
    __shared__ float sh_m[kRowWaves];
    const int64_t row = blockIdx.y;
    if (!live(a, row)) return;
    const auto* z = reinterpret_cast<const typename E::S*>(a.logits) + row / a.W * a.ld_seq + row % a.W * a.ld_beam;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int per = (a.segs + a.chunks - 1) / a.chunks, s0 = blockIdx.x * per, s1 = s0 + per < a.segs ? s0 + per : a.segs;
    float m = -INFINITY;
    double sum = 0.0;
    for (int s = s0 + w; s < s1; s += kRowWaves) {
        float x[E::V];
        load_logits<DT>(z, (int64_t)s * SEG + lane * E::V, a.V, x);
        float top = x[0];
#pragma unroll
        for (int j = 1; j < E::V; ++j) top = fmaxf(top, x[j]);
        top = wave_max(top);
        if (lane == 0) a.seg_max[row * a.segs + s] = top;
        if (top > m) {
            if (m != -INFINITY) sum *= exp((double)m - (double)top);
            m = top;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < E::V; ++j) part += exp_diff(x[j], ref);
        sum += part;
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

struct Chosen {
    uint64_t key[kMaxCount];
    int id[kMaxCount];
    int n;
};
struct Scratch {
    uint64_t list_key[kList];
    int list_id[kList];
    int bins[kBins];
    uint64_t hi, lo;
    int above, inside, listed, wave[kSelThreads / 64];
};

// The workgroup's reduction of two 64-bit numbers: largest and smallest.
__device__ __forceinline__ void wave_range(uint64_t& hi, uint64_t& lo) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t h = __shfl_xor((unsigned long long)hi, o, 64), l = __shfl_xor((unsigned long long)lo, o, 64);
        hi = h > hi ? h : hi;
        lo = l < lo ? l : lo;
    }
}

// The K items of largest key among i < n, equal keys by the smaller id, best first, into
// `out`.  item(i, key, id) is false for one that is none.  The interval [lo, hi] of keys in
// which the K-th lies is cut into 2048 bins, again and again, until what lies at or above
// it fits the list; keys that are all equal are cut by their ids instead.
template <class F>
__device__ void select(int64_t n, int K, F item, Scratch& s, Chosen& out) {
    const int t = threadIdx.x;
    __syncthreads();
    if (t == 0) { s.hi = 0; s.lo = ~0ull; s.inside = 0; s.above = 0; s.listed = 0; }
    __syncthreads();
    uint64_t hi = 0, lo = ~0ull;
    int count = 0;
    for (int64_t i = t; i < n; i += kSelThreads) {
        uint64_t key;
        int id;
        if (!item(i, key, id)) continue;
        hi = key > hi ? key : hi;
        lo = key < lo ? key : lo;
        ++count;
    }
    wave_range(hi, lo);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) count += __shfl_xor(count, o, 64);
    if ((t & 63) == 0 && count) {
        atomicMax((unsigned long long*)&s.hi, (unsigned long long)hi);
        atomicMin((unsigned long long*)&s.lo, (unsigned long long)lo);
        atomicAdd(&s.inside, count);
    }
    __syncthreads();
    bool by_id = false;
    uint64_t tied = 0;
    // (6 cuts of 11 bits end the keys, 3 the ids)
    for (int cut = 0; cut < 12 && s.above + s.inside > kList; ++cut) {
        const uint64_t H = s.hi, L = s.lo;
        if (H == L && !by_id) {   // (ids are distinct, so this happens once)
            by_id = true;
            tied = H;
            __syncthreads();
            if (t == 0) { s.hi = 0xffffffffull; s.lo = 0; }
            __syncthreads();
            continue;
        }
        int shift = 0;
        while ((H - L) >> shift >= kBins) ++shift;
        const int above = s.above;
        for (int i = t; i < kBins; i += kSelThreads) s.bins[i] = 0;
        __syncthreads();
        for (int64_t i = t; i < n; i += kSelThreads) {
            uint64_t key;
            int id;
            if (!item(i, key, id)) continue;
            if (by_id) {
                if (key != tied) continue;
                key = 0xffffffffull - (uint32_t)id;   // the smaller id first
            }
            if (key >= L && key <= H) atomicAdd(&s.bins[(H - key) >> shift], 1);
        }
        __syncthreads();
        // the bin in which the count passes K: each thread two bins, summed over waves
        const int b0 = s.bins[2 * t], b1 = s.bins[2 * t + 1];
        int before = b0 + b1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(before, o, 64);
            if ((t & 63) >= o) before += x;
        }
        if ((t & 63) == 63) s.wave[t >> 6] = before;
        __syncthreads();
        for (int i = 0; i < (t >> 6); ++i) before += s.wave[i];
        before += above - b0 - b1;   // items of bins before this thread's, and above all
        int bin = -1, first = 0, in = 0;
        if (before < K && before + b0 >= K) { bin = 2 * t; first = before; in = b0; }
        else if (before + b0 < K && before + b0 + b1 >= K) { bin = 2 * t + 1; first = before + b0; in = b1; }
        if (bin >= 0) {
            const uint64_t nh = H - ((uint64_t)bin << shift);
            const uint64_t width = ((uint64_t)1 << shift) - 1;
            s.hi = nh;
            s.lo = nh - L > width ? nh - width : L;
            s.above = first;
            s.inside = in;
        }
        __syncthreads();
    }
    const uint64_t L = s.lo;
    for (int64_t i = t; i < n; i += kSelThreads) {
        uint64_t key;
        int id;
        if (!item(i, key, id)) continue;
        const bool in = by_id ? key > tied || (key == tied && 0xffffffffull - (uint32_t)id >= L) : key >= L;
        if (in) {
            const int at = atomicAdd(&s.listed, 1);
            if (at < kList) {
                s.list_key[at] = key;
                s.list_id[at] = id;
            }
        }
    }
    __syncthreads();
    const int m = s.listed < kList ? s.listed : kList;
    if (t < m) {
        const uint64_t key = s.list_key[t];
        const int id = s.list_id[t];
        int rank = 0;
        for (int i = 0; i < m; ++i) rank += s.list_key[i] > key || (s.list_key[i] == key && s.list_id[i] < id);
        if (rank < K) { out.key[rank] = key; out.id[rank] = id; }
    }
    if (t == 0) out.n = m < K ? m : K;
    __syncthreads();
}

// One workgroup a sequence.
template <int DT>
__global__ __launch_bounds__(kSelThreads) void beam_select_kernel(BeamArgs a) {
    using E = Elem<DT>;
    constexpr int SEG = 64 * E::V;
    __shared__ double score[kMaxBeams], log_sum[kMaxBeams];   // a beam that has ended: log_sum = NaN
    __shared__ float largest[kMaxBeams];
    __shared__ Scratch scratch;
    __shared__ Chosen segs, best;
    __shared__ int bad;
    const int64_t g = blockIdx.x, row0 = g * a.W;
    const int lane = threadIdx.x & 63, t = threadIdx.x;
    if (t == 0) bad = 0;
    __syncthreads();
    for (int w = t >> 6; w < a.W; w += kSelThreads / 64) {
        const float c = a.scores[row0 + w];
        double l = NAN, m = -INFINITY;
        if (live(a, row0 + w)) {
            double sum = 0.0;
            for (int i = lane; i < a.chunks; i += 64) m = fmax(m, a.part[(row0 + w) * a.chunks + i].x);
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) m = fmax(m, __shfl_xor(m, o, 64));
            for (int i = lane; i < a.chunks; i += 64) {
                const double2 p = a.part[(row0 + w) * a.chunks + i];
                sum += p.x == m ? p.y : p.y * exp(p.x - m);
            }
            sum = wave_sum(sum);
            l = m == -INFINITY && sum == 0.0 ? 0.0 : log(sum);   // nothing but -inf: no candidates
            if (lane == 0 && l != l) bad = 1;                    // +inf among the logits: inf - inf
        }
        if (lane == 0) {
            score[w] = c;
            largest[w] = (float)m;
            log_sum[w] = l;
            if (!(c < INFINITY)) bad = 1;
        }
    }
    __syncthreads();
    if (bad) {
        for (int r = t; r < a.count; r += kSelThreads) {
            a.out_scores[g * a.count + r] = NAN;
            a.parents[g * a.count + r] = a.tokens[g * a.count + r] = 0;
        }
        return;
    }
    // the best segments; of an ended beam its first stands for the end
    select((int64_t)a.W * a.segs, a.count, [&](int64_t i, uint64_t& key, int& id) {
        const int w = (int)(i / a.segs), sg = (int)(i - (int64_t)w * a.segs);
        if (score[w] == -INFINITY) return false;
        id = (int)i;
        if (log_sum[w] != log_sum[w]) {
            key = key_of(score[w]);
            return sg == 0;
        }
        const float z = a.seg_max[(row0 + w) * a.segs + sg];
        key = key_of(score[w] + (((double)z - largest[w]) - log_sum[w]));
        return z != -INFINITY;
    }, scratch, segs);
    // their candidates, none worse than the last segment's best where there are enough
    const uint64_t least = segs.n == a.count ? segs.key[segs.n - 1] : 0;
    const auto* z0 = reinterpret_cast<const typename E::S*>(a.logits) + g * a.ld_seq;
    select((int64_t)segs.n * SEG, a.count, [&](int64_t i, uint64_t& key, int& id) {
        const int sg = segs.id[i / SEG], w = sg / a.segs;
        int j = (sg - w * a.segs) * SEG + (int)(i % SEG);
        if (log_sum[w] != log_sum[w]) {
            if (i % SEG) return false;
            key = key_of(score[w]);
            id = w * a.V + (int)a.end;
            return true;
        }
        if (j >= a.V) return false;
        const float z = E::to_f(z0[w * a.ld_beam + j]);
        key = key_of(score[w] + (((double)z - largest[w]) - log_sum[w]));
        id = w * a.V + j;
        return z != -INFINITY && key >= least;
    }, scratch, best);
    for (int r = t; r < a.count; r += kSelThreads) {
        const bool some = r < best.n;
        a.out_scores[g * a.count + r] = some ? (float)value_of(best.key[r]) : -INFINITY;
        a.parents[g * a.count + r] = some ? best.id[r] / a.V : 0;
        a.tokens[g * a.count + r] = some ? best.id[r] % a.V : 0;
    }
}

int segment(int dtype) { return 64 * (dtype == AXS6_F32 ? 4 : 8); }
int64_t segments(int64_t V, int dtype) { return (V + segment(dtype) - 1) / segment(dtype); }
// Workgroups a row: four segments a wave, or fewer where the rows are few.
int64_t chunks_of(int64_t rows, int64_t segs) {
    int64_t per = 16 * kRowWaves;
    while (per > kRowWaves && rows * ((segs + per - 1) / per) < 1024) per /= 2;
    return (segs + per - 1) / per;
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int64_t axs6_beam_select_workspace(int64_t G, int64_t W, int64_t V, int32_t dtype) {
    if (G <= 0 || W <= 0 || V <= 0 || !valid_dtype(dtype)) return 0;
    const int64_t segs = segments(V, dtype);
    return G * W * (chunks_of(G * W, segs) * (int64_t)sizeof(double2) + (segs + 3) / 4 * 16);
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
    const int64_t need = axs6_beam_select_workspace(G, W, V, dtype);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: a 16-byte aligned workspace of %lld bytes required, got %lld", fn,
                    (long long)need, (long long)workspace_bytes);
    BeamArgs a{};
    a.logits = logits; a.ld_seq = ld_sequence; a.ld_beam = ld_beam; a.scores = scores; a.finished = finished; a.end = end;
    a.W = (int)W; a.V = (int)V; a.count = (int)count;
    a.segs = (int)segments(V, dtype); a.chunks = (int)chunks_of(G * W, a.segs);
    a.part = reinterpret_cast<double2*>(workspace);
    a.seg_max = reinterpret_cast<float*>(a.part + G * W * a.chunks);
    a.out_scores = out_scores; a.parents = parents; a.tokens = tokens;
    const dim3 grid((unsigned)a.chunks, (unsigned)(G * W));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == AXS6_F32) {
        beam_rows_kernel<AXS6_F32><<<grid, 64 * kRowWaves, 0, st>>>(a);
        beam_select_kernel<AXS6_F32><<<(unsigned)G, kSelThreads, 0, st>>>(a);
    } else if (dtype == AXS6_BF16) {
        beam_rows_kernel<AXS6_BF16><<<grid, 64 * kRowWaves, 0, st>>>(a);
        beam_select_kernel<AXS6_BF16><<<(unsigned)G, kSelThreads, 0, st>>>(a);
    } else {
        beam_rows_kernel<AXS6_F16><<<grid, 64 * kRowWaves, 0, st>>>(a);
        beam_select_kernel<AXS6_F16><<<(unsigned)G, kSelThreads, 0, st>>>(a);
    }
    return check_launch(fn);
}
