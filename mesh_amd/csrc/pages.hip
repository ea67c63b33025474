// Pages of the KV pool copied inside it: a fork's first write into a page that
// another session still reads (copy on write), and a compaction's moves.
// No counterpart in the reference, whose sessions never share pages
// (DeviceLayerKVCache owns its pages, forward_pass.rs:250-460).
//
//   pool[l][dst_i] = pool[l][src_i] for every layer l
//
// Bound by HBM: each page is read once and written once (1025 pages of 64 KiB in
// 32 layers: 838 us, 5.13 TB/s, as a large copy; 15 pages of 16 KiB in 22: a launch).
#include "zr_internal.h"

namespace zr {

// Pairs travel as a kernel argument (at most 4 KiB of them): nothing is staged,
// so the call returns with its arrays free and later calls share no buffer.  A
// few (a fork's first writes) go as a small one, which costs the host less.
constexpr int kPairsPerLaunch = 448, kFewPairs = 32;
template <int N> struct PagePairs {
    int src[N], dst[N];
};

// A workgroup copies 16 KiB of one pair's page in one layer: 4 loads of 16 B
// per lane go out together.  Block b is chunk b % chunks of pair b / chunks.
constexpr int kCopyVecs = 4;
constexpr int kCopyChunk = 256 * kCopyVecs * 16;  // bytes

template <int N>
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(unsigned char* pool, size_t layer_bytes, uint32_t page_bytes,
                                                            int chunks, PagePairs<N> pp) {
    const int pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks;
    unsigned char* layer = pool + (size_t)blockIdx.y * layer_bytes;
    const uint4* src = (const uint4*)(layer + (size_t)pp.src[pair] * page_bytes);
    uint4* dst = (uint4*)(layer + (size_t)pp.dst[pair] * page_bytes);
    const uint32_t vecs = page_bytes / 16, v0 = (uint32_t)chunk * (256 * kCopyVecs) + threadIdx.x;
    uint4 x[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
        if (v0 + 256 * i < vecs) x[i] = src[v0 + 256 * i];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
        if (v0 + 256 * i < vecs) dst[v0 + 256 * i] = x[i];
}

template <int N> static void launch_pairs(zr_context* ctx, const int* src, const int* dst, int m) {
    // a page is 2 kv_cols x 16 elements, kv_cols a multiple of 4: whole 16-byte vectors
    const int chunks = (int)((ctx->page_bytes + kCopyChunk - 1) / kCopyChunk);
    PagePairs<N> pp;
    for (int j = 0; j < N; ++j) {  // (past m: never read)
        pp.src[j] = j < m ? src[j] : 0;
        pp.dst[j] = j < m ? dst[j] : 0;
    }
    hipLaunchKernelGGL(kv_copy_pages_kernel<N>, dim3(m * chunks, ctx->desc.num_layers), dim3(256), 0, ctx->stream,
                       (unsigned char*)ctx->kv_pool, ctx->page_bytes * ctx->n_pages, (uint32_t)ctx->page_bytes, chunks, pp);
}

zr_status launch_kv_copy_pages(zr_context* ctx, const int* src, const int* dst, int n) {
    if (n <= 0) return ZR_OK;
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassOther, &ev);
    for (int i = 0; i < n; i += kPairsPerLaunch) {
        const int m = std::min(kPairsPerLaunch, n - i);
        if (m <= kFewPairs) launch_pairs<kFewPairs>(ctx, src + i, dst + i, m); else launch_pairs<kPairsPerLaunch>(ctx, src + i, dst + i, m);
        ZR_LAUNCH_CHECK(ctx);
    }
    timing_mark_end(ctx, kClassOther, ev);
    return ZR_OK;
}

}  // namespace zr
