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
// Bound by HBM: each source is read and each target written once.
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

// One workgroup a (group, head) and every gridDim.y-th piece of its places.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_copy_kernel(CopyArgs a) {
    extern __shared__ int sh[];            // each target's source, or -1, and its length
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
        from[i] = n > 0 ? (int)p : -1;
        len[i] = (int)n;
        if (n > 0) atomicMax(&top, (int)n);
    }
    __syncthreads();
    const int cols = 1 << a.cols_log2, blocks = (top + kKvBlock - 1) / kKvBlock;
    // pieces of the six tensors: 16-byte values of codes and tails, 4-byte ones of scales
    const int block_vecs = kKvBlock * a.D / 16, row_vecs = a.D * a.es / 16;
    const int64_t code_pieces = ((int64_t)blocks * block_vecs + cols - 1) >> a.cols_log2;
    const int scale_pieces = (blocks + cols - 1) >> a.cols_log2, tail_pieces = (kKvBlock * row_vecs + cols - 1) >> a.cols_log2;
    const int64_t pieces = 2 * (code_pieces + scale_pieces + tail_pieces);
    if (blocks == 0) return;
    const int items = a.W << a.cols_log2;
    for (int64_t piece = blockIdx.y; piece < pieces; piece += gridDim.y) {
        int z;                       // which tensor
        int64_t at = piece;          // which piece of it
        if (at < 2 * code_pieces) { z = at < code_pieces ? 0 : 2; at -= z ? code_pieces : 0; }
        else if ((at -= 2 * code_pieces) < 2 * scale_pieces) { z = at < scale_pieces ? 1 : 3; at -= z == 3 ? scale_pieces : 0; }
        else { at -= 2 * scale_pieces; z = at < tail_pieces ? 4 : 5; at -= z == 5 ? tail_pieces : 0; }
        const int64_t c0 = at << a.cols_log2;
        const bool scales = z == 1 || z == 3, tail = z >= 4;
        // values of a sequence's head in the cache and in the target
        const int64_t per_src = scales ? a.nb_src : tail ? kKvBlock * row_vecs : (int64_t)a.nb_src * block_vecs;
        const int64_t per_dst = scales ? a.nb_dst : tail ? kKvBlock * row_vecs : (int64_t)a.nb_dst * block_vecs;
        u32x4 v[kItems];
        int64_t to[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int item = threadIdx.x + k * THREADS, i = item >> a.cols_log2;
            const int64_t c = c0 + (item & (cols - 1));
            to[k] = -1;
            v[k] = u32x4{0, 0, 0, 0};
            if (item >= items) continue;
            const int p = from[i];
            if (p < 0) continue;
            const int n = len[i], nb = (n + kKvBlock - 1) / kKvBlock;
            const int64_t count = scales ? nb : tail ? n % kKvBlock * row_vecs : (int64_t)nb * block_vecs;
            if (c >= count) continue;
            to[k] = ((g * a.dst_seq + w0 + i) * a.H + h) * per_dst + c;
            const int64_t s = ((g * a.src_seq + p) * a.H + h) * per_src + c;
            if (scales) v[k].x = reinterpret_cast<const uint32_t*>(a.src[z])[s];
            else v[k] = reinterpret_cast<const u32x4*>(a.src[z])[s];
        }
        if (a.in_place) {
            // the values are here before any of them is written over
#pragma unroll
            for (int k = 0; k < kItems; ++k) asm volatile("" : "+v"(v[k]));
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if (to[k] < 0) continue;
            if (scales) reinterpret_cast<uint32_t*>(a.dst[z])[to[k]] = v[k].x;
            else reinterpret_cast<u32x4*>(a.dst[z])[to[k]] = v[k];
        }
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
    while (a.cols_log2 < 10 && (a.W << (a.cols_log2 + 1)) <= kItems * threads) ++a.cols_log2;
    const int64_t tiles = (targets + a.W - 1) / a.W;
    if (tiles > 65535) return fail(AXS6_ERR_INVALID_ARGUMENT, "%s: dimension too large", fn);
    const int64_t nb = blocks < target_blocks ? blocks : target_blocks;
    int64_t pieces = (2 * (nb * kKvBlock * D / 16 + nb) >> a.cols_log2) + 4;
    const int64_t want = (4096 + groups * H * tiles - 1) / (groups * H * tiles);
    if (pieces > want) pieces = want;
    if (pieces > 65535) pieces = 65535;
    const dim3 grid((unsigned)(groups * H), (unsigned)pieces, (unsigned)tiles);
    const size_t lds = 2 * a.W * sizeof(int);
    hipStream_t st = (hipStream_t)stream;
    if (threads == 256) kv_copy_kernel<256><<<grid, 256, lds, st>>>(a);
    else kv_copy_kernel<1024><<<grid, 1024, lds, st>>>(a);
    return check_launch(fn);
}
