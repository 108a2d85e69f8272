// Sequences of the 8-bit cache copied: beams after their parents, a prompt forked,
// finished sequences closed up.
//
// Sequence i of the target becomes sequence src(i) of the cache, its first n tokens,
// n that sequence's length: ceil(n / 32) blocks of codes and scales, and the n % 32 raw
// rows of a partial block.  Nothing else of the target is written.  In place every
// target may be another one's source, so a workgroup reads what all sequences of a
// group have in the same places, waits, and writes: no order of the sequences is
// needed and no second buffer.
//
// Bound by HBM: each source is read and each target written once.  Measured: 32 groups of
// 8 beams, 2047 tokens, 8 heads of 128 (950 MB) in 208 us, 4.6 TB/s; 256 sequences of 375
// to 1500 tokens closed up, 4 heads of 64 (200 MB), in 43 us, 4.7 TB/s; a prompt of 4001
// tokens forked 8 ways for 8 groups, 12 heads of 80, in 66 us; four beams of 40 tokens in
// 4 us, of which the launch and the chain sources - lengths - codes are all.
//
// - A head's blocks lie behind one another in both caches, so a piece is one run of 16-byte
//   places and a thread keeps the same sequences through all its pieces: what remains a
//   piece is a load, in place a barrier, and a store.  (Finding tensor, sequence and length
//   anew for each value: 96 us for the 256 sequences.)
// - A workgroup takes 1024 threads where a group is so large that fewer would leave a
//   sequence less than a cache line of a piece (256 sequences closed up 42 us, with 256 threads 58, 1000 of them 202
//   and 729; 17 sequences 7.7, with 1024 8.2).  Two of 1024 or eight of 256 fit a CU; calls
//   of few pieces start just as many workgroups as fit (1 x 134 sequences of 288 tokens:
//   8.8 us, one workgroup a piece 12.0), those of more than 12 times as
//   many pieces four times that, so that the last ones to end are short (32 x 8 beams: 208 us, as many as fit 238; from 3
//   times as many on, 256 sequences closed up 42 -> 47, from 48, the beams 238).
// - Stores pass the L2 by: what a fork reads stays there for its other sequences (95 us
//   without, for 66; beams 219 for 214, closing up 45 for 43).
// - Loading the next piece before this one is stored was slower at all sizes (43 to 48 us
//   for the 256 sequences, 214 to 225 us for the beams): the workgroups beside it do that.
#include "axs6_internal.h"
#include "kv_cache.h"
#include "nf5_device.h"

namespace axs6 {
namespace {

constexpr int kItems = 4;              // values a thread holds between reading and writing
constexpr int kTile = AXS6_KV_COPY_MAX_IN_PLACE;   // values a workgroup of 1024 threads holds
static_assert(kTile == kItems * 1024);

struct CopyArgs {
    const void* src[6];        // key codes and scales, value codes and scales, tails
    void* dst[6];
    const int64_t *sources, *lengths;
    int64_t src_seq, dst_seq;  // sequences a group has in the cache, and in the target
    int W;                     // of the target's, those a workgroup takes: in place all
    int H, D, nb_src, nb_dst, es;
    int cols_log2;             // places of all W sequences that a workgroup takes at once
    int in_place;
};

// A thread's part of every piece: the same place of kItems of the target's sequences.
struct Item {
    uint32_t src, dst;         // sequences' heads in the cache and in the target
    int n;                     // tokens
};

// In place: all threads' values are here before any place is written.
template <class T>
__device__ __forceinline__ void arrived(T (&v)[kItems], int in_place) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) asm volatile("" : "+v"(v[k]) : : "memory");
    if (in_place) __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

// One workgroup a (group, head) and every gridDim.y-th piece of its places.
template <int THREADS>
__global__ __launch_bounds__(THREADS, 8) void kv_copy_kernel(CopyArgs a) {
    extern __shared__ int sh[];            // each target's source, and its length, 0 where nothing is copied
    __shared__ int top;
    int *from = sh, *len = sh + a.W;
    const int g = blockIdx.x / a.H, h = blockIdx.x % a.H;
    const int64_t w0 = (int64_t)blockIdx.z * a.W;
    const int64_t cap = (int64_t)(a.nb_src < a.nb_dst ? a.nb_src : a.nb_dst) * kKvBlock;
    if (threadIdx.x == 0) top = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.W; i += THREADS) {
        const int64_t p = w0 + i < a.dst_seq ? a.sources[g * a.dst_seq + w0 + i] : -1;
        const bool use = p >= 0 && p < a.src_seq && !(a.in_place && p == i);
        int64_t n = use ? a.lengths[g * a.src_seq + p] : 0;
        n = n < 0 ? 0 : n > cap ? cap : n;
        from[i] = use ? (int)p : 0;
        len[i] = (int)n;
        if (n > 0) atomicMax(&top, (int)n);
    }
    __syncthreads();
    const int blocks = (top + kKvBlock - 1) / kKvBlock, block_vecs = kKvBlock * a.D / 16, row_vecs = a.D * a.es / 16;
    if (blocks == 0) return;
    const int cols = 1 << a.cols_log2, col = threadIdx.x & (cols - 1);
    Item it[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int i = (threadIdx.x + k * THREADS) >> a.cols_log2;
        const bool in = i < a.W;
        it[k].n = in ? len[i] : 0;
        it[k].src = (uint32_t)((g * a.src_seq + (in ? from[i] : 0)) * a.H + h);
        it[k].dst = (uint32_t)((g * a.dst_seq + w0 + i) * a.H + h);
    }

    // codes: a head's blocks lie behind one another; pieces of keys and of values take turns
    const int pieces = 2 * ((blocks * block_vecs + cols - 1) >> a.cols_log2);
    const uint32_t per_src = (uint32_t)(a.nb_src * block_vecs), per_dst = (uint32_t)(a.nb_dst * block_vecs);
    auto has = [&](int p, int k) { return (p >> 1 << a.cols_log2) + col < (it[k].n + kKvBlock - 1) / kKvBlock * block_vecs; };
    const int step = gridDim.y;
    int p = blockIdx.y;
    for (; p < pieces; p += step) {
        const int64_t at = (p >> 1 << a.cols_log2) + col;
        const u32x4* src = reinterpret_cast<const u32x4*>(a.src[p & 1 ? 2 : 0]) + at;
        u32x4* dst = reinterpret_cast<u32x4*>(a.dst[p & 1 ? 2 : 0]) + at;
        u32x4 v[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            v[k] = u32x4{0, 0, 0, 0};
            if (has(p, k)) v[k] = src[(uint64_t)it[k].src * per_src];
        }
        arrived(v, a.in_place);
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (has(p, k)) __builtin_nontemporal_store(v[k], dst + (uint64_t)it[k].dst * per_dst);
    }

    // scales and raw rows: more pieces behind those of the codes
    const int scale_pieces = 2 * ((blocks + cols - 1) >> a.cols_log2), tail_pieces = 2 * ((kKvBlock * row_vecs + cols - 1) >> a.cols_log2);
    for (p -= pieces; p < scale_pieces; p += step) {
        const int c = (p >> 1 << a.cols_log2) + col, z = p & 1 ? 3 : 1;
        uint32_t v[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            v[k] = 0;
            if (c * kKvBlock < it[k].n) v[k] = reinterpret_cast<const uint32_t*>(a.src[z])[(uint64_t)it[k].src * (uint32_t)a.nb_src + c];
        }
        arrived(v, a.in_place);
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (c * kKvBlock < it[k].n) reinterpret_cast<uint32_t*>(a.dst[z])[(uint64_t)it[k].dst * (uint32_t)a.nb_dst + c] = v[k];
    }
    for (p -= scale_pieces; p < tail_pieces; p += step) {
        const int c = (p >> 1 << a.cols_log2) + col, z = p & 1 ? 5 : 4;
        u32x4 v[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            v[k] = u32x4{0, 0, 0, 0};
            if (c < it[k].n % kKvBlock * row_vecs) v[k] = reinterpret_cast<const u32x4*>(a.src[z])[(uint64_t)it[k].src * (kKvBlock * row_vecs) + c];
        }
        arrived(v, a.in_place);
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (c < it[k].n % kKvBlock * row_vecs) reinterpret_cast<u32x4*>(a.dst[z])[(uint64_t)it[k].dst * (kKvBlock * row_vecs) + c] = v[k];
    }
}

}  // namespace
}  // namespace axs6

using namespace axs6;

extern "C" int axs6_kv_copy(const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales,
                            const void* k_tail, const void* v_tail, int32_t dtype, int64_t groups, int64_t sequences,
                            int64_t targets, int64_t H, int64_t D, int64_t blocks, const int64_t* sources,
                            const int64_t* lengths, int64_t target_blocks, void* k_codes_out, float* k_scales_out,
                            void* v_codes_out, float* v_scales_out, void* k_tail_out, void* v_tail_out, void* stream) {
    const char* fn = "axs6_kv_copy";
    if (!valid_dtype(dtype)) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: unknown dtype code %d", fn, dtype);
    if (groups < 0 || sequences < 0 || targets < 0 || groups > ((int64_t)1 << 31) - 1 || sequences > ((int64_t)1 << 31) - 1 ||
        targets > ((int64_t)1 << 31) - 1)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: bad number of sequences", fn);
    int rc = check_cache(fn, groups * sequences, H, D, blocks, k_codes, k_scales, v_codes, v_scales);
    if (rc) return rc;
    rc = check_cache(fn, groups * targets, H, D, target_blocks, k_codes_out, k_scales_out, v_codes_out, v_scales_out);
    if (rc) return rc;
    if (groups * sequences * targets * H * blocks * target_blocks == 0) return AXS6_OK;
    if (!sources || !lengths || !k_tail || !v_tail || !k_tail_out || !v_tail_out)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: null sources, lengths or tail", fn);
    if (((uintptr_t)k_tail | (uintptr_t)v_tail | (uintptr_t)k_tail_out | (uintptr_t)v_tail_out) % 16)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: tails not aligned to 16 bytes", fn);
    CopyArgs a{};
    const void* src[6] = {k_codes, k_scales, v_codes, v_scales, k_tail, v_tail};
    void* dst[6] = {k_codes_out, k_scales_out, v_codes_out, v_scales_out, k_tail_out, v_tail_out};
    // in place: all six tensors are the cache's own; else none may share memory with it
    const int64_t es = dtype == AXS6_F32 ? 4 : 2;
    int same = 0, overlap = 0;
    for (int i = 0; i < 6; ++i) {
        a.src[i] = src[i];
        a.dst[i] = dst[i];
        same += src[i] == dst[i];
        for (int j = 0; j < 6; ++j) {
            auto bytes = [&](int k, int64_t n, int64_t nb) {
                return n * H * (k >= 4 ? kKvBlock * D * es : nb * (k % 2 ? 4 : kKvBlock * D));
            };
            const uintptr_t s = (uintptr_t)src[i], d = (uintptr_t)dst[j];
            if (s < d + bytes(j, groups * targets, target_blocks) && d < s + bytes(i, groups * sequences, blocks))
                overlap += !(i == j && s == d);
        }
    }
    a.in_place = same == 6 && sequences == targets && blocks == target_blocks;
    if (overlap || (same && !a.in_place))
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: the target shares memory with the cache without being it", fn);
    if (a.in_place && targets > kTile)
        return fail(AXS6_ERR_UNSUPPORTED, "%s: at most %d sequences a group in place, got %lld", fn, kTile, (long long)targets);
    if (groups * H > ((int64_t)1 << 31) - 1) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    a.sources = sources; a.lengths = lengths; a.src_seq = sequences; a.dst_seq = targets;
    a.W = (int)(a.in_place || targets < 64 ? targets : 64);
    a.H = (int)H; a.D = (int)D; a.nb_src = (int)blocks; a.nb_dst = (int)target_blocks; a.es = (int)es;
    const int threads = a.W <= 64 ? 256 : 1024;
    while ((2 << a.cols_log2) <= threads && (a.W << (a.cols_log2 + 1)) <= kItems * threads) ++a.cols_log2;
    const int64_t tiles = (targets + a.W - 1) / a.W, nb = blocks < target_blocks ? blocks : target_blocks;
    // a piece's places are counted in 32 bits, and a sequence's head's
    if (tiles > 65535 || (blocks > target_blocks ? blocks : target_blocks) * (2 * D) >= (int64_t)1 << 30)
        return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    int64_t pieces = (2 * (nb * kKvBlock * D / 16 + nb) >> a.cols_log2) + 4;
    const int64_t heads = groups * H * tiles, fit = 512 * 1024 / threads, want = pieces * heads > 12 * fit ? 4 * fit : fit;
    if (pieces * heads > want) pieces = (want + heads - 1) / heads;
    if (pieces > 65535) pieces = 65535;
    const dim3 grid((unsigned)(groups * H), (unsigned)pieces, (unsigned)tiles);
    const size_t lds = 2 * a.W * sizeof(int);
    hipStream_t st = (hipStream_t)stream;
    if (threads == 256) kv_copy_kernel<256><<<grid, 256, lds, st>>>(a);
    else kv_copy_kernel<1024><<<grid, 1024, lds, st>>>(a);
    return check_launch(fn);
}
