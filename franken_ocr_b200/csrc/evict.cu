// Eviction from a paged K/V cache by accumulated attention weight.
//
// A row of n entries shrinks to `budget`: the first `sink` and the last
// `recent` entries stay, and of those between them the budget - sink - recent
// with the largest weights (equal weights: the lower position).  Each kv head
// chooses for itself.  What is kept moves, in order, to pages of its own, so
// pages shared with other rows are never written.
//
// evict_select_kernel finds the threshold weight by a radix descent over the
// weights' ordered bit patterns and writes the kept positions in order;
// evict_gather_kernel copies their K, V and weights.
#include "paged.cuh"

namespace focr {
namespace {

constexpr int SEL = 1024;

// Unsigned integers that order like the weights: -0 equals 0, NaN lies below
// every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct EvictArgs {
    PagedView c;
    const int32_t *into;   // new page lists
    const int32_t *lens;
    const float *w;
    float *w_out;
    int32_t *kept, *lens_out;
    long long w_row, w_head, into_stride;
    int rows, width, budget, sink, recent, into_pages;
};

// The row's length; one that passes its weights or its pages counts as 0.
__device__ __forceinline__ int evict_len(const EvictArgs &a, int r) {
    const int n = a.lens[r];
    return n < 0 || n > a.width || n > a.c.max_pages * a.c.page_size ? 0 : n;
}

__global__ void __launch_bounds__(SEL) evict_select_kernel(const EvictArgs a) {
    __shared__ int hist[256], wsum[2][32], found[2], base[2];
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.y, h = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int n = evict_len(a, r);
    int32_t *kept = a.kept + ((int64_t)r * a.c.kv_heads + h) * a.budget;
    if (t == 0 && h == 0) a.lens_out[r] = min(n, a.budget);
    if (n <= a.budget) {
        for (int i = t; i < a.budget; i += SEL) kept[i] = i < n ? i : -1;
        return;
    }
    const float *w = a.w + r * a.w_row + h * a.w_head;
    const int lo = a.sink, hi = n - a.recent, want = a.budget - a.sink - a.recent;
    uint32_t prefix = 0, mask = 0;
    int left = want;   // how many of the entries that match the prefix are kept
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = t; i < 256; i += SEL) hist[i] = 0;
            __syncthreads();
            for (int i = lo + t; i < hi; i += SEL) {
                const uint32_t k = weight_key(w[i]);
                if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255], 1);
            }
            __syncthreads();
            if (t == 0) {
                int above = 0, b = 255;
                while (above + hist[b] < left) above += hist[b--];
                found[0] = b;
                found[1] = left - above;
            }
            __syncthreads();
            prefix |= (uint32_t)found[0] << shift;
            mask |= 255u << shift;
            left = found[1];
            __syncthreads();
        }
    }
    // entries above `prefix` stay, and the first `left` of those equal to it
    if (t == 0) base[0] = base[1] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += SEL) {
        const int i = i0 + t;
        bool keep = false, tie = false;
        if (i < n) {
            if (i < lo || i >= hi) keep = true;
            else if (want > 0) {
                const uint32_t k = weight_key(w[i]);
                keep = k > prefix;
                tie = k == prefix;
            }
        }
        const unsigned ties = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) wsum[0][warp] = __popc(ties);
        __syncthreads();
        int before = base[0] + __popc(ties & ((1u << lane) - 1));
        for (int x = 0; x < warp; x++) before += wsum[0][x];
        if (tie && before < left) keep = true;
        const unsigned keeps = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) wsum[1][warp] = __popc(keeps);
        __syncthreads();
        int at = base[1] + __popc(keeps & ((1u << lane) - 1));
        for (int x = 0; x < warp; x++) at += wsum[1][x];
        if (keep) kept[at] = i;
        __syncthreads();
        if (t == 0)
            for (int x = 0; x < 32; x++) {
                base[0] += wsum[0][x];
                base[1] += wsum[1][x];
            }
        __syncthreads();
    }
}

// A thread per 16-byte chunk of a kept entry; then the weights with zeros
// behind the kept ones.
__global__ void __launch_bounds__(256) evict_gather_kernel(const EvictArgs a) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, h = blockIdx.y;
    const int n = evict_len(a, r), live = min(n, a.budget);
    const int32_t *kept = a.kept + ((int64_t)r * a.c.kv_heads + h) * a.budget;
    const int cpr = a.c.row_bytes / 16;
    const int32_t *from = a.c.table + r * a.c.table_stride, *to = a.into + r * a.into_stride;
    PagedView dst = a.c;
    for (unsigned x = blockIdx.x * 256 + threadIdx.x; x < (unsigned)(live * cpr); x += gridDim.x * 256) {
        const unsigned j = x / cpr, ch = x - j * cpr;
        const int64_t s = a.c.offset(from, (uint32_t)kept[j]), d = dst.offset(to, (uint32_t)j);
        if (s < 0 || d < 0) continue;
        const int64_t o = h * a.c.head_stride + ch * 16;
        *(uint4 *)(a.c.k + d + o) = *(const uint4 *)(a.c.k + s + o);
        *(uint4 *)(a.c.v + d + o) = *(const uint4 *)(a.c.v + s + o);
    }
    const float *w = a.w + r * a.w_row + h * a.w_head;
    float *wo = a.w_out + ((int64_t)r * a.c.kv_heads + h) * a.width;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < a.width; i += gridDim.x * 256)
        wo[i] = i < live ? w[kept[i]] : 0.0f;
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" int focr_paged_evict(const focr_paged_cache *cache, size_t rows, const int32_t *lens,
                                const float *weights, size_t width, size_t weights_row_stride,
                                size_t weights_head_stride, const int32_t *new_table,
                                size_t new_table_stride, size_t new_pages, size_t budget,
                                size_t sink, size_t recent, int32_t *kept, int32_t *lens_out,
                                float *weights_out, void *stream) {
    return guarded("paged_evict", [&]() -> int {
        EvictArgs a{};
        int rc = paged_view("paged_evict", cache, rows, &a.c);
        if (rc) return rc;
        if (budget == 0 || sink > budget || recent > budget - sink)
            return fail(FOCR_E_SHAPE, "paged_evict: sink " + std::to_string(sink) + " + recent " +
                                          std::to_string(recent) + " over budget " +
                                          std::to_string(budget));
        if (rows == 0) return FOCR_OK;
        if (!lens || !weights || !new_table || !kept || !lens_out || !weights_out)
            return fail(FOCR_E_ARG, "paged_evict: null pointer");
        if (rows > 65535 || cache->kv_heads > 65535 || budget > (size_t)INT32_MAX / 64 ||
            width > INT32_MAX || new_pages > INT32_MAX)
            return fail(FOCR_E_UNSUPPORTED, "paged_evict: dimension out of range");
        if (width == 0 || (cache->kv_heads > 1 && weights_head_stride < width) ||
            (rows > 1 && weights_row_stride < width))
            return fail(FOCR_E_SHAPE, "paged_evict: a weights stride is shorter than the width");
        if ((uint64_t)new_pages * cache->page_size < budget ||
            (rows > 1 && new_table_stride < new_pages))
            return fail(FOCR_E_SHAPE, "paged_evict: the new pages hold fewer entries than the budget");
        if (lens_out == lens)
            return fail(FOCR_E_ARG, "paged_evict: lens_out must not be lens");
        if (weights_out == weights)
            return fail(FOCR_E_ARG, "paged_evict: weights_out must not be weights");
        if (new_table == cache->table)
            return fail(FOCR_E_ARG, "paged_evict: the new pages must not be the old ones");
        a.into = new_table;
        a.lens = lens;
        a.w = weights;
        a.w_out = weights_out;
        a.kept = kept;
        a.lens_out = lens_out;
        a.w_row = (long long)weights_row_stride;
        a.w_head = (long long)weights_head_stride;
        a.into_stride = (long long)new_table_stride;
        a.rows = (int)rows;
        a.width = (int)width;
        a.budget = (int)budget;
        a.sink = (int)sink;
        a.recent = (int)recent;
        a.into_pages = (int)new_pages;
        cudaStream_t st = (cudaStream_t)stream;
        FOCR_CUDA_TRY(launch_pdl(evict_select_kernel, dim3(cache->kv_heads, (unsigned)rows), SEL, 0, st, a));
        const size_t n = budget * (a.c.row_bytes / 16), most = n > width ? n : width;
        const unsigned blocks = (unsigned)((most + 1023) / 1024);
        FOCR_CUDA_TRY(launch_pdl(evict_gather_kernel, dim3(blocks < 256 ? blocks : 256, cache->kv_heads, (unsigned)rows),
                                 256, 0, st, a));
        return FOCR_OK;
    });
}
