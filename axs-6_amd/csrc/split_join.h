// Joining a row's partial attention results: the keys were split over
// workgroups, each of which left its sums of D values, its maximum and its sum of
// exponentials (in units of log2).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace axs6 {
namespace {

constexpr int kMaxSplits = 128;    // of one row
constexpr int kJoinThreads = 256;  // one workgroup a row
typedef float join4 __attribute__((ext_vector_type(4)));

struct Joined {
    join4 o;       // values d .. d + 3 of the row's sums
    float m, l;    // its maximum and sum
    int d;         // below 0 in threads that have none
};

// part: (splits, rows, D), stat: (splits, rows, 2); D a multiple of 4, up to 256.  A
// thread has one split's factor; groups of D / 4 threads take every so-many-th
// split's sums, which are added in order.
__device__ __forceinline__ Joined join_row(const float* part, const float* stat, int64_t rows, int64_t row, int splits,
                                           int D) {
    __shared__ float factor[kMaxSplits], red[2][kJoinThreads / 64];
    __shared__ __attribute__((aligned(16))) join4 sums[kJoinThreads];
    const int i = threadIdx.x, w = i >> 6;
    float m = -INFINITY, l = 0.0f;
    if (i < splits) {
        const float2 st = *reinterpret_cast<const float2*>(stat + 2 * (i * rows + row));
        m = st.x;
        l = st.y;
    }
    Joined r;
    r.m = m;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, o, 64));
    if ((i & 63) == 0) red[0][w] = r.m;
    __syncthreads();
    r.m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float f = __builtin_amdgcn_exp2f(m - (r.m == -INFINITY ? 0.0f : r.m));
    if (i < kMaxSplits) factor[i] = f;
    l *= f;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
    if ((i & 63) == 0) red[1][w] = l;
    __syncthreads();
    r.l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const int lanes = D / 4, groups = kJoinThreads / lanes, g = i / lanes;
    r.d = i % lanes * 4;
    r.o = join4{0.0f, 0.0f, 0.0f, 0.0f};
    if (g < groups) {
#pragma unroll 4
        for (int s = g; s < splits; s += groups)
            r.o += *reinterpret_cast<const join4*>(part + (s * rows + row) * D + r.d) * factor[s];
        sums[i] = r.o;
    }
    __syncthreads();
    if (g != 0) {
        r.d = -1;
        return r;
    }
    for (int j = 1; j < groups; ++j) r.o += sums[j * lanes + i];
    return r;
}

// The same for few splits of many rows: a thread has four values of one row and
// walks over its splits; thread i of all.
constexpr int kFewSplits = 8;
// A workgroup a row takes 22 us for 16000 rows of 3 splits, this form 8; for 256
// rows of 2 it is the other way round, 2 us against 4.
inline bool join_by_value(int64_t rows, int splits) { return splits <= kFewSplits && rows >= 1024; }
__device__ __forceinline__ Joined join_few(const float* part, const float* stat, int64_t rows, int64_t i, int splits,
                                           int D, int64_t& row) {
    const int lanes = D / 4;
    row = i / lanes;
    Joined r{join4{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f, -1};
    if (row >= rows) return r;
    r.d = (int)(i - row * lanes) * 4;
    float2 st[kFewSplits];
    join4 x[kFewSplits];
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        st[s] = make_float2(-INFINITY, 0.0f);
        x[s] = join4{0.0f, 0.0f, 0.0f, 0.0f};
        if (s < splits) {
            st[s] = *reinterpret_cast<const float2*>(stat + 2 * (s * rows + row));
            x[s] = *reinterpret_cast<const join4*>(part + (s * rows + row) * D + r.d);
        }
        r.m = fmaxf(r.m, st[s].x);
    }
    const float ref = r.m == -INFINITY ? 0.0f : r.m;
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        if (s >= splits) continue;
        const float f = __builtin_amdgcn_exp2f(st[s].x - ref);
        r.l += st[s].y * f;
        r.o += x[s] * f;
    }
    return r;
}

}  // namespace
}  // namespace axs6
