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
#include <cooperative_groups.h>

#include <algorithm>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace focr {
namespace {

constexpr int SEL = 1024;              // threads of a select block
constexpr int BINS = 2048;
constexpr int HELD = 40960;            // weights a block keeps in shared memory

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

// One cluster a (row, head): every block takes an equal run of the positions
// between sink and recent, reads its weights once and keeps their keys.  Three
// passes of 11, 11 and 10 bits narrow the threshold; the blocks' histograms meet
// in block 0's shared memory.  It ends early when a whole bin stays.  Then the
// kept positions of each run are counted, and written behind those of the runs
// before.
__global__ void __launch_bounds__(SEL) evict_select_kernel(const EvictArgs a, int held) {
    extern __shared__ uint32_t keys[];   // held
    __shared__ int hist[BINS], counts[2], before[2], wsum[2][32], chosen[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), size = (int)cluster.num_blocks();
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, h = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int n = evict_len(a, r);
    int32_t *kept = a.kept + ((int64_t)r * a.c.kv_heads + h) * a.budget;
    if (t == 0 && h == 0 && rank == 0) a.lens_out[r] = min(n, a.budget);
    if (n <= a.budget) {
        for (int i = rank * SEL + t; i < a.budget; i += size * SEL) kept[i] = i < n ? i : -1;
        return;
    }
    const float *w = a.w + r * a.w_row + h * a.w_head;
    const int lo = a.sink, hi = n - a.recent, want = a.budget - a.sink - a.recent;
    for (int i = rank * SEL + t; i < a.sink; i += size * SEL) kept[i] = i;
    for (int i = rank * SEL + t; i < a.recent; i += size * SEL) kept[a.sink + want + i] = hi + i;
    if (want == 0) return;   // the same for the whole cluster
    const int per = (hi - lo + size - 1) / size;
    const int begin = min(hi, lo + rank * per), end = min(hi, begin + per), m = end - begin;
    for (int i = t; i < min(m, held); i += SEL) keys[i] = weight_key(w[begin + i]);
    auto key = [&](int i) { return i < held ? keys[i] : weight_key(w[begin + i]); };

    uint32_t prefix = 0;
    int left = want, shift = 32;   // `left` of the keys that match `prefix` above `shift` stay
    bool all = false;              // all of them do
    int *hist0 = cluster.map_shared_rank(hist, 0);
#pragma unroll 1
    for (int pass = 0; pass < 3 && !all; pass++) {
        const int bits = pass < 2 ? 11 : 10, next = shift - bits;
        for (int i = t; i < BINS; i += SEL) hist[i] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < m; i0 += SEL) {
            const int i = i0 + t;
            const uint32_t k = i < m ? key(i) : 0;
            const bool in = i < m && (pass == 0 || k >> shift == prefix >> shift);
            const int bin = in ? (int)(k >> next & ((1u << bits) - 1)) : -1;
            // many equal weights (all that was never looked at) would queue up
            int same;
            __match_all_sync(0xffffffffu, bin, &same);
            if (same) {
                if (in && lane == 0) atomicAdd(&hist[bin], 32);
            } else if (in) {
                atomicAdd(&hist[bin], 1);
            }
        }
        if (size > 1) {
            cluster.sync();
            if (rank)
                for (int i = t; i < BINS; i += SEL)
                    if (hist[i]) atomicAdd(&hist0[i], hist[i]);
            cluster.sync();
        } else {
            __syncthreads();
        }
        // the bin in which the `left`-th largest lies: counts from the top
        constexpr int PER = BINS / SEL;
        const int top = (1 << bits) - 1 - t * PER;   // this thread's bins, downwards
        int c[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            c[i] = top - i >= 0 ? hist0[top - i] : 0;
            sum += c[i];
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) wsum[0][warp] = inc;
        __syncthreads();
        int above = inc - sum;
        for (int x = 0; x < warp; x++) above += wsum[0][x];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (above < left && above + c[i] >= left) {
                chosen[0] = top - i;
                chosen[1] = (left - above) | (c[i] == left - above ? 1 << 30 : 0);
            }
            above += c[i];
        }
        if (size > 1) cluster.sync();   // block 0's bins have been read
        else __syncthreads();
        prefix |= (uint32_t)chosen[0] << next;
        left = chosen[1] & ~(1 << 30);
        all = chosen[1] >> 30;
        shift = next;
        __syncthreads();
    }
    // larger keys stay, and of the equal ones all or the first `left`.  Each warp
    // has a run of its own, so the order is the positions'.
    const uint32_t limit = prefix >> shift;
    const int each = ((m + SEL - 1) / SEL) * 32, w0 = min(m, warp * each), w1 = min(m, w0 + each);
    int larger = 0, equal = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t k = key(i) >> shift;
        larger += k > limit;
        equal += k == limit;
    }
    larger = __reduce_add_sync(0xffffffffu, larger);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        wsum[0][warp] = larger;
        wsum[1][warp] = equal;
    }
    __syncthreads();
    if (warp < 2) {   // prefix over the warps, and the block's total
        const int x = wsum[warp][lane];
        int inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        wsum[warp][lane] = inc - x;
        if (lane == 31) counts[warp] = inc;
    }
    __syncthreads();
    if (size > 1) {
        cluster.sync();
        if (t < 2) {
            int x = 0;
            for (int b = 0; b < rank; b++) x += cluster.map_shared_rank(counts, b)[t];
            before[t] = x;
        }
        cluster.sync();   // and nobody leaves while its counts are read
    } else {
        if (t < 2) before[t] = 0;
        __syncthreads();
    }
    int L = before[0] + wsum[0][warp], E = before[1] + wsum[1][warp];
    kept += a.sink;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t k = i < w1 ? key(i) >> shift : 0;
        const bool gt = i < w1 && k > limit, eq = i < w1 && k == limit;
        const unsigned gts = __ballot_sync(0xffffffffu, gt), eqs = __ballot_sync(0xffffffffu, eq);
        const unsigned below = (1u << lane) - 1;
        const int e = E + __popc(eqs & below);
        if (gt || (eq && (all || e < left)))
            kept[L + __popc(gts & below) + (all ? e : min(e, left))] = begin + i;
        L += __popc(gts);
        E += __popc(eqs);
    }
}

// A thread per 16-byte chunk of U kept entries at a time (position, page and chunk
// are loads that wait for one another, so several chains run side by side);
// then the weights, with zeros behind the kept ones.
__global__ void __launch_bounds__(256) evict_gather_kernel(const EvictArgs a) {
    constexpr int U = 4;
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, h = blockIdx.y;
    const int n = evict_len(a, r), live = min(n, a.budget);
    const int32_t *kept = a.kept + ((int64_t)r * a.c.kv_heads + h) * a.budget;
    const unsigned cpr = a.c.row_bytes / 16, total = (unsigned)live * cpr;
    const int32_t *from = a.c.table + r * a.c.table_stride, *to = a.into + r * a.into_stride;
    const char *kb = a.c.k + h * a.c.head_stride, *vb = a.c.v + h * a.c.head_stride;
    for (unsigned x0 = blockIdx.x * (256 * U) + threadIdx.x; x0 < total; x0 += gridDim.x * (256 * U)) {
        int pos[U];
        int64_t s[U], d[U];
        uint4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const unsigned x = x0 + u * 256;
            pos[u] = x < total ? kept[x / cpr] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const unsigned x = x0 + u * 256, j = x / cpr;
            s[u] = d[u] = -1;
            if (pos[u] >= 0) {
                s[u] = a.c.offset(from, (uint32_t)pos[u]);
                d[u] = a.c.offset(to, j);
            }
            if (d[u] < 0) s[u] = -1;
            s[u] += s[u] < 0 ? 0 : (int64_t)(x - j * cpr) * 16;
            d[u] += (int64_t)(x - j * cpr) * 16;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (s[u] >= 0) {
                k[u] = *(const uint4 *)(kb + s[u]);
                v[u] = *(const uint4 *)(vb + s[u]);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (s[u] >= 0) {
                *(uint4 *)(const_cast<char *>(kb) + d[u]) = k[u];
                *(uint4 *)(const_cast<char *>(vb) + d[u]) = v[u];
            }
    }
    const float *w = a.w + r * a.w_row + h * a.w_head;
    float *wo = a.w_out + ((int64_t)r * a.c.kv_heads + h) * a.width;
    for (int i0 = blockIdx.x * (256 * U) + threadIdx.x; i0 < a.width; i0 += gridDim.x * (256 * U)) {
        int pos[U];
        float y[U];
#pragma unroll
        for (int u = 0; u < U; u++) pos[u] = i0 + u * 256 < live ? kept[i0 + u * 256] : -1;
#pragma unroll
        for (int u = 0; u < U; u++) y[u] = pos[u] >= 0 ? w[pos[u]] : 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u * 256 < a.width) wo[i0 + u * 256] = y[u];
    }
}

// Blocks of a cluster: enough that each has at most 4096 of the weights a row may
// have, 8 at most.
int select_blocks(size_t width) {
    int n = 1;
    while (n < 8 && (size_t)n * 4096 < width) n <<= 1;
    return n;
}

int launch_select(const EvictArgs &a, cudaStream_t st) {
    const int size = select_blocks((size_t)a.width);
    const int held = (int)std::min<size_t>(HELD, ((size_t)a.width + size - 1) / size);
    FOCR_CUDA_TRY(set_max_dynamic_smem((const void *)evict_select_kernel, HELD * 4));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size, a.c.kv_heads, a.rows);
    cfg.blockDim = SEL;
    cfg.dynamicSmemBytes = (size_t)held * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    FOCR_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_select_kernel, a, held));
    return FOCR_OK;
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
            width > (1u << 30) || new_pages > INT32_MAX)
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
        if ((rc = launch_select(a, st))) return rc;
        const size_t n = budget * (a.c.row_bytes / 16), most = n > width ? n : width;
        const unsigned blocks = (unsigned)((most + 1023) / 1024);
        FOCR_CUDA_TRY(launch_pdl(evict_gather_kernel, dim3(blocks < 256 ? blocks : 256, cache->kv_heads, (unsigned)rows),
                                 256, 0, st, a));
        return FOCR_OK;
    });
}
