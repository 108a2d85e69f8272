// Distillation from a teacher's top logits: the loss of each row and the
// gradient of the student's logits.
//
// Row r has student logits z[V] and the teacher's K top logits t with their
// classes idx; T is the temperature.  Over the K entries with idx >= 0
//   p_k = softmax(t / T)_k,  log q_j = z_j / T - lse,  lse = log sum_j exp(z_j / T),
//   loss_r = T^2 sum_k p_k (log p_k - log q_idx_k)          (a term with p_k = 0 is 0),
//   dloss_r / dz_j = T (q_j - sum of p_k over the k with idx_k = j)   (0 without entries),
// and the loss is sum_r w_r loss_r, over sum_r w_r for the mean.  A row of
// weight 0 is not read.  A class at or past V gives the row NaN.
//
// Bound by HBM: the forward reads the logits once (running maximum and sum of
// exponentials in one pass), the backward reads them and writes the gradient
// once; the K entries of a row are gathered from cache.  All sums are float32
// in a fixed order; the gradient is rounded once.
// A class may stand in several entries: the backward compares a row's entries with each
// other, K^2 of them, which is nothing for a teacher's top logits and much for whole
// vocabularies (2048 x 32000 bf16, the backward: K = 64 75 us, 512 317, 2048
// 4.0 ms; 256 x 32000, K = 32000: 193 ms).
// The gradient could only be written by the forward if its factor from above
// were known there, or by a second rounding: so three passes, 6 bytes a logit.
// Measured: 8192 x 128000 bf16, both directions, 1206 us, 5.2 TB/s over the three
// passes (two read 2.1 GB, one writes it); 509 x 1000 float32 63 us, of which the
// caller's backward call is nearly all.
#include <math.h>

#include "axs6_internal.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

constexpr int kDistillThreads = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DistillArgs {
    const void* logits;
    int64_t ld, N, V;
    const float* values;
    const int64_t* indices;
    int64_t K;
    float T;
    const float* weights;
    float *rows, *stats;        // loss of each row; its largest logit and 1 / sum exp((z - largest) / T)
    const float* grad_out;      // one value, or one a row (grad_rows)
    const float* norm;          // factor of every row's gradient, or null
    void* dz;
    int grad_rows;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The reduction of `v` over the workgroup; every thread gets it.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const float w = __shfl_xor(v, o, 64);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    __syncthreads();   // red may still be read by the previous reduction
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < kDistillThreads / 64; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
    return v;
}

// max(a, b) that keeps a NaN of either, which fmaxf drops.
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }

// m, l: the running maximum of x and the sum of exp2((x - m) c) so far.  The
// maximum is subtracted before the factor log2(e) / T: the values that carry
// the sum lie near it, where the difference is exact.
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2, float c) {
    const float n = max_nan(m, m2);
    const float ref = n == -INFINITY ? 0.0f : n;
    l = l * exp2_fast((m - ref) * c) + l2 * exp2_fast((m2 - ref) * c);
    m = n;
}

// The teacher's softmax over its entries: maximum and sum of exponentials; the
// sum is 0 where no entry counts.
__device__ __forceinline__ void teacher(const DistillArgs& a, int64_t r, float* red, float& tm, float& tl) {
    const float c = kLog2e / a.T;
    float m = -INFINITY;
    for (int64_t k = threadIdx.x; k < a.K; k += kDistillThreads)
        if (a.indices[r * a.K + k] >= 0) m = fmaxf(m, a.values[r * a.K + k]);
    tm = block_reduce<true>(m, red);
    const float ref = tm == -INFINITY ? 0.0f : tm;
    float l = 0.0f;
    for (int64_t k = threadIdx.x; k < a.K; k += kDistillThreads)
        if (a.indices[r * a.K + k] >= 0) l += exp2_fast((a.values[r * a.K + k] - ref) * c);
    tl = block_reduce<false>(l, red);
    tm = ref;
}

// One workgroup a row.
template <int DT, bool VEC>
__global__ __launch_bounds__(kDistillThreads) void distill_forward_kernel(DistillArgs a) {
    using E = Elem<DT>;
    __shared__ float red[kDistillThreads / 64], red2[kDistillThreads / 64];
    const int64_t r = blockIdx.x;
    if (a.weights && a.weights[r] == 0.0f) {
        if (threadIdx.x == 0) { a.rows[r] = 0.0f; a.stats[2 * r] = 0.0f; a.stats[2 * r + 1] = 0.0f; }
        return;
    }
    const auto* z = reinterpret_cast<const typename E::S*>(a.logits) + r * a.ld;
    const float c = kLog2e / a.T;
    constexpr int W = VEC ? E::V : 1;
    float m = -INFINITY, l = 0.0f;
    for (int64_t i = (int64_t)threadIdx.x * W; i < a.V; i += (int64_t)kDistillThreads * W) {
        float x[W];
        if constexpr (VEC) E::unpack(*reinterpret_cast<const u32x4*>(z + i), x);
        else x[0] = E::to_f(z[i]);
        float n = m;
#pragma unroll
        for (int j = 0; j < W; ++j) n = max_nan(n, x[j]);
        const float ref = n == -INFINITY ? 0.0f : n;
        float s = l * exp2_fast((m - ref) * c);
#pragma unroll
        for (int j = 0; j < W; ++j) s += exp2_fast((x[j] - ref) * c);
        m = n;
        l = s;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) join(m, l, __shfl_xor(m, o, 64), __shfl_xor(l, o, 64), c);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = m; red2[threadIdx.x >> 6] = l; }
    __syncthreads();
    m = red[0]; l = red2[0];
#pragma unroll
    for (int i = 1; i < kDistillThreads / 64; ++i) join(m, l, red[i], red2[i], c);
    const float logl = __builtin_amdgcn_logf(l);   // log2, as every exponent here
    float tm, tl;
    teacher(a, r, red, tm, tl);
    const float logtl = __builtin_amdgcn_logf(tl);
    float sum = 0.0f;
    for (int64_t k = threadIdx.x; k < a.K; k += kDistillThreads) {
        const int64_t j = a.indices[r * a.K + k];
        if (j < 0) continue;
        const float lp = (a.values[r * a.K + k] - tm) * c - logtl;
        const float p = exp2_fast(lp);
        if (j >= a.V) sum = __uint_as_float(0x7fc00000u);
        else if (!(p == 0.0f)) sum += p * (lp - ((E::to_f(z[j]) - m) * c - logl));
    }
    sum = block_reduce<false>(sum, red);
    if (threadIdx.x == 0) {
        a.rows[r] = tl == 0.0f ? 0.0f : a.T * a.T * kLn2 * sum;
        a.stats[2 * r] = m;
        a.stats[2 * r + 1] = 1.0f / l;
    }
}

// loss[0] = sum w l, over sum w for the mean; norm[0] = 1 or 1 / sum w (0 where
// the weights sum to 0).  One workgroup, a fixed order.
__global__ __launch_bounds__(kDistillThreads) void distill_sum_kernel(const float* rows, const float* weights,
                                                                      int64_t N, int mean, float* loss, float* norm) {
    __shared__ float red[kDistillThreads / 64];
    float s = 0.0f, w = 0.0f;
    // eight loads on their way at once: one by one 8192 rows took 16 us
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < N; i += kDistillThreads) {
        const float wi = weights ? weights[i] : 1.0f, ri = rows[i];
        s += wi != 0.0f ? wi * ri : 0.0f;
        w += wi;
    }
    s = block_reduce<false>(s, red);
    w = block_reduce<false>(w, red);
    if (threadIdx.x == 0) {
        const float f = !mean ? 1.0f : w == 0.0f ? 0.0f : 1.0f / w;
        loss[0] = !mean ? s : w == 0.0f ? 0.0f : s / w;
        norm[0] = f;
    }
}

// One workgroup a row: the dense gradient first, then the K classes again with
// the teacher's probabilities (of repeated classes each writes the same sum).
template <int DT, bool VEC>
__global__ __launch_bounds__(kDistillThreads) void distill_backward_kernel(DistillArgs a) {
    using E = Elem<DT>;
    __shared__ float red[kDistillThreads / 64];
    const int64_t r = blockIdx.x;
    constexpr int W = VEC ? E::V : 1;
    auto* dz = reinterpret_cast<typename E::S*>(a.dz) + r * a.V;
    const float w = a.weights ? a.weights[r] : 1.0f;
    float tm = 0.0f, tl = 0.0f;
    if (w != 0.0f) teacher(a, r, red, tm, tl);
    if (w == 0.0f || tl == 0.0f) {   // a row of no weight or without entries
        float zero[W] = {};
        for (int64_t i = (int64_t)threadIdx.x * W; i < a.V; i += (int64_t)kDistillThreads * W) {
            if constexpr (VEC) *reinterpret_cast<u32x4*>(dz + i) = E::pack(zero);
            else dz[i] = E::from_f(0.0f);
        }
        return;
    }
    const auto* z = reinterpret_cast<const typename E::S*>(a.logits) + r * a.ld;
    const float c = kLog2e / a.T, m = a.stats[2 * r], rl = a.stats[2 * r + 1], rtl = 1.0f / tl;
    const float f = a.T * w * a.grad_out[a.grad_rows ? r : 0] * (a.norm ? a.norm[0] : 1.0f);
    bool bad = false;
    for (int64_t k = threadIdx.x; k < a.K; k += kDistillThreads) bad = bad || a.indices[r * a.K + k] >= a.V;
    const float g = __syncthreads_or(bad) ? __uint_as_float(0x7fc00000u) : f;
    const float gl = g * rl;
    for (int64_t i = (int64_t)threadIdx.x * W; i < a.V; i += (int64_t)kDistillThreads * W) {
        float x[W];
        if constexpr (VEC) E::unpack(*reinterpret_cast<const u32x4*>(z + i), x);
        else x[0] = E::to_f(z[i]);
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = gl * exp2_fast((x[j] - m) * c);
        if constexpr (VEC) *reinterpret_cast<u32x4*>(dz + i) = E::pack(x);
        else dz[i] = E::from_f(x[0]);
    }
    __syncthreads();   // the dense values are written before those of the K classes
    for (int64_t k = threadIdx.x; k < a.K; k += kDistillThreads) {
        const int64_t j = a.indices[r * a.K + k];
        if (j < 0 || j >= a.V) continue;
        float p = 0.0f;
        for (int64_t o = 0; o < a.K; ++o)
            if (a.indices[r * a.K + o] == j) p += exp2_fast((a.values[r * a.K + o] - tm) * c);
        dz[j] = E::from_f(g * (exp2_fast((E::to_f(z[j]) - m) * c) * rl - p * rtl));
    }
}

int check_common(const char* fn, const void* logits, int dtype, int64_t ld, int64_t N, int64_t V, const float* values,
                 const int64_t* indices, int64_t K, float T) {
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    if (N < 0 || V < 0 || K < 0 || N > ((int64_t)1 << 31) - 1 || V > ((int64_t)1 << 40) || K > ((int64_t)1 << 31))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: negative or too large a dimension", fn);
    if (!(T > 0.0f) || !isfinite(T))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: the temperature must be positive and finite", fn);
    if (N && V && (!logits || ld < V)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null logits or rows that overlap", fn);
    if (N && K && (!values || !indices)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null teacher logits", fn);
    if ((uintptr_t)logits % (dtype == AXS6_F32 ? 4 : 2))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not element-aligned", fn);
    return AXS6_OK;
}

// Whether every row is whole aligned 16-byte vectors.
bool whole_vectors(int dtype, int64_t ld, int64_t V, const void* a, const void* b) {
    const int64_t v = dtype == AXS6_F32 ? 4 : 8;
    return V % v == 0 && ld % v == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0;
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int axs6_distill_forward(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V,
                                    const float* values, const int64_t* indices, int64_t K, float temperature,
                                    const float* weights, int32_t mean, float* rows, float* stats, float* loss,
                                    float* norm, void* stream) {
    const char* fn = "axs6_distill_forward";
    int rc = check_common(fn, logits, dtype, ld, N, V, values, indices, K, temperature);
    if (rc) return rc;
    if ((N && (!rows || !stats)) || (loss && !norm)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null output", fn);
    DistillArgs a{};
    a.logits = logits; a.ld = ld; a.N = N; a.V = V; a.values = values; a.indices = indices; a.K = K;
    a.T = temperature; a.weights = weights; a.rows = rows; a.stats = stats;
    hipStream_t st = (hipStream_t)stream;
    if (N) {
        const bool vec = whole_vectors(dtype, ld, V, logits, nullptr);
        const unsigned n = (unsigned)N;
        switch (dtype * 2 + vec) {
            case AXS6_F32 * 2: distill_forward_kernel<AXS6_F32, false><<<n, kDistillThreads, 0, st>>>(a); break;
            case AXS6_F32 * 2 + 1: distill_forward_kernel<AXS6_F32, true><<<n, kDistillThreads, 0, st>>>(a); break;
            case AXS6_BF16 * 2: distill_forward_kernel<AXS6_BF16, false><<<n, kDistillThreads, 0, st>>>(a); break;
            case AXS6_BF16 * 2 + 1: distill_forward_kernel<AXS6_BF16, true><<<n, kDistillThreads, 0, st>>>(a); break;
            case AXS6_F16 * 2: distill_forward_kernel<AXS6_F16, false><<<n, kDistillThreads, 0, st>>>(a); break;
            default: distill_forward_kernel<AXS6_F16, true><<<n, kDistillThreads, 0, st>>>(a); break;
        }
    }
    if (loss) distill_sum_kernel<<<1, kDistillThreads, 0, st>>>(rows, weights, N, mean, loss, norm);
    return check_launch(fn);
}

extern "C" int axs6_distill_backward(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V,
                                     const float* values, const int64_t* indices, int64_t K, float temperature,
                                     const float* weights, const float* stats, const float* grad_out,
                                     int32_t grad_rows, const float* norm, void* dlogits, void* stream) {
    const char* fn = "axs6_distill_backward";
    int rc = check_common(fn, logits, dtype, ld, N, V, values, indices, K, temperature);
    if (rc) return rc;
    if (N == 0 || V == 0) return AXS6_OK;
    if (!stats || !grad_out || !dlogits) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null statistics, gradient or output", fn);
    if ((uintptr_t)dlogits % (dtype == AXS6_F32 ? 4 : 2))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: pointer not element-aligned", fn);
    DistillArgs a{};
    a.logits = logits; a.ld = ld; a.N = N; a.V = V; a.values = values; a.indices = indices; a.K = K;
    a.T = temperature; a.weights = weights; a.stats = const_cast<float*>(stats); a.grad_out = grad_out;
    a.grad_rows = grad_rows; a.norm = norm; a.dz = dlogits;
    hipStream_t st = (hipStream_t)stream;
    const bool vec = whole_vectors(dtype, ld, V, logits, dlogits);
    const unsigned n = (unsigned)N;
    switch (dtype * 2 + vec) {
        case AXS6_F32 * 2: distill_backward_kernel<AXS6_F32, false><<<n, kDistillThreads, 0, st>>>(a); break;
        case AXS6_F32 * 2 + 1: distill_backward_kernel<AXS6_F32, true><<<n, kDistillThreads, 0, st>>>(a); break;
        case AXS6_BF16 * 2: distill_backward_kernel<AXS6_BF16, false><<<n, kDistillThreads, 0, st>>>(a); break;
        case AXS6_BF16 * 2 + 1: distill_backward_kernel<AXS6_BF16, true><<<n, kDistillThreads, 0, st>>>(a); break;
        case AXS6_F16 * 2: distill_backward_kernel<AXS6_F16, false><<<n, kDistillThreads, 0, st>>>(a); break;
        default: distill_backward_kernel<AXS6_F16, true><<<n, kDistillThreads, 0, st>>>(a); break;
    }
    return check_launch(fn);
}
