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

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace focr {
namespace {

constexpr int SEL = 512;      // threads of a select block
constexpr int HELD = 40;      // most keys of a thread that shared memory holds
constexpr int BINS = 2048;
constexpr int MOST = 8;       // blocks of a cluster
constexpr uint32_t ZERO = 0x80000000u;   // the key of weight 0
constexpr uint32_t LOST = 0x7fff7fffu;   // one NaN of f32, two of f16 or bf16

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
    int width, budget, sink, recent;
};

// The row's length; one that passes its weights or its pages counts as 0.
__device__ __forceinline__ int evict_len(const EvictArgs &a, int r) {
    const int n = a.lens[r];
    return n < 0 || n > a.width || n > a.c.max_pages * a.c.page_size ? 0 : n;
}

// One cluster a (row, head): every warp takes an equal run of the positions
// between sink and recent, reads its weights once and keeps their keys in shared
// memory.  Three passes of 11, 11 and 10 bits narrow the threshold, fewer where
// a whole bin stays; after each the blocks add up a share of the bins each and
// hand the sums to all.  Then the kept positions of each run are counted, and
// written behind those of the runs before.
//
// The weights are a hundredth of the bytes that the gather moves: instructions and
// the barriers bound it, so zeros (all that was never looked at) are counted by
// vote and not one by one, and equal weights are told apart only where the
// threshold falls among them.  16 rows and heads of 131072 weights: 25 us; 160 of up
// to 4097: 11 us.
__global__ void __launch_bounds__(SEL, 2) evict_select_kernel(const EvictArgs a, int held) {
    extern __shared__ uint32_t keys[];   // [held steps][SEL], a warp's run together
    __shared__ int hist[BINS], totals[2][BINS];
    __shared__ int counts[2], before[2], wsum[2][SEL / 32], chosen[2];
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
    // this warp's run: [run, run + 32 steps), of which `mine` are this lane's
    const int steps = (hi - lo + size * SEL - 1) / (size * SEL);
    const int run = lo + (rank * (SEL / 32) + warp) * 32 * steps;
    const int mine = run + lane < hi ? min(steps, (hi - run - lane + 31) >> 5) : 0;
    w += run + lane;
    const int near = min(steps, held);
    uint32_t *own = keys + warp * 32 * near + lane;
    // f(step, key, whether there is one) for every step, the warp together
    auto every = [&](auto f) {
#pragma unroll 4
        for (int k = 0; k < near; k++) f(k, own[32 * k], k < mine);
#pragma unroll 1
        for (int k = near; k < steps; k++) f(k, k < mine ? weight_key(w[32ll * k]) : 0, k < mine);
    };

    uint32_t prefix = 0;
    int left = want, shift = 32;   // `left` of the keys that match `prefix` above `shift` stay
    bool all = false;              // all of them do
#pragma unroll 1
    for (int pass = 0; pass < 3 && !all; pass++) {
        const int bits = pass < 2 ? 11 : 10, next = shift - bits;
        for (int i = t; i < BINS; i += SEL) hist[i] = 0;
        __syncthreads();
        int zeros = 0;
        if (pass == 0) {
            constexpr int U = 8;
            for (int k0 = 0; k0 < steps; k0 += U) {
                float x[U];
#pragma unroll
                for (int u = 0; u < U; u++) x[u] = k0 + u < mine ? w[32ll * (k0 + u)] : 0.0f;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const bool have = k0 + u < mine;
                    const uint32_t k = weight_key(x[u]);
                    if (k0 + u < near) own[32 * (k0 + u)] = k;
                    zeros += __popc(__ballot_sync(0xffffffffu, have && k == ZERO));
                    if (have && k != ZERO) atomicAdd(&hist[k >> 21], 1);
                }
            }
        } else {
            const uint32_t match = prefix >> shift;
            const bool with_zero = match == ZERO >> shift;
            if (with_zero)
                every([&](int, uint32_t x, bool have) {
                    zeros += __popc(__ballot_sync(0xffffffffu, have && x == ZERO));
                    if (have && x >> shift == match && x != ZERO) atomicAdd(&hist[x >> next & ((1u << bits) - 1)], 1);
                });
            else
                every([&](int, uint32_t x, bool have) {
                    if (have && x >> shift == match) atomicAdd(&hist[x >> next & ((1u << bits) - 1)], 1);
                });
        }
        if (lane == 0 && zeros) atomicAdd(&hist[ZERO >> next & ((1u << bits) - 1)], zeros);
        int *total = hist;
        if (size > 1) {
            total = totals[pass & 1];   // the other one may still be read
            cluster.sync();
            const int share = BINS / size;
            for (int i = t; i < share; i += SEL) {
                const int bin = rank * share + i;
                int x[MOST], sum = 0;
#pragma unroll
                for (int q = 0; q < MOST; q++) x[q] = q < size ? cluster.map_shared_rank(hist, q)[bin] : 0;
#pragma unroll
                for (int q = 0; q < MOST; q++) sum += x[q];
#pragma unroll
                for (int q = 0; q < MOST; q++)
                    if (q < size) cluster.map_shared_rank(total, q)[bin] = sum;
            }
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
            c[i] = top - i >= 0 ? total[top - i] : 0;
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
#pragma unroll
        for (int x = 0; x < SEL / 32; x++) above += x < warp ? wsum[0][x] : 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (above < left && above + c[i] >= left) {
                chosen[0] = top - i;
                chosen[1] = (left - above) | (c[i] == left - above ? 1 << 30 : 0);
            }
            above += c[i];
        }
        __syncthreads();
        prefix |= (uint32_t)chosen[0] << next;
        left = chosen[1] & ~(1 << 30);
        all = chosen[1] >> 30;
        shift = next;
        __syncthreads();
    }
    // larger keys stay, and of the equal ones all or the first `left`
    const uint32_t limit = prefix >> shift, over = all ? limit : limit + 1;
    int larger = 0, equal = 0;
    every([&](int, uint32_t k, bool have) {
        const uint32_t x = k >> shift;
        larger += have && x >= over;
        equal += have && x == limit;
    });
    larger = __reduce_add_sync(0xffffffffu, larger);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        wsum[0][warp] = larger;
        wsum[1][warp] = equal;
    }
    __syncthreads();
    if (warp < 2) {   // prefix over the warps, and the block's total
        const int x = lane < SEL / 32 ? wsum[warp][lane] : 0;
        int inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane < SEL / 32) wsum[warp][lane] = inc - x;
        if (lane == 31) counts[warp] = inc;
    }
    __syncthreads();
    if (size > 1) {
        cluster.sync();
        if (warp < 2) {
            int x = lane < rank ? cluster.map_shared_rank(counts, lane)[warp] : 0;
            x = __reduce_add_sync(0xffffffffu, x);
            if (lane == 0) before[warp] = x;
        }
        cluster.sync();   // and nobody leaves while its counts are read
    } else {
        if (t < 2) before[t] = 0;
        __syncthreads();
    }
    int L = before[0] + wsum[0][warp], E = before[1] + wsum[1][warp];
    kept += a.sink;
    const unsigned below = (1u << lane) - 1;
    if (all) {
        every([&](int step, uint32_t k, bool have) {
            const bool in = have && k >> shift >= limit;
            const unsigned ins = __ballot_sync(0xffffffffu, in);
            if (in) kept[L + __popc(ins & below)] = run + 32 * step + lane;
            L += __popc(ins);
        });
        return;
    }
    every([&](int step, uint32_t k, bool have) {
        const uint32_t x = k >> shift;
        const bool gt = have && x > limit, eq = have && x == limit;
        const unsigned gts = __ballot_sync(0xffffffffu, gt), eqs = __ballot_sync(0xffffffffu, eq);
        const int e = E + __popc(eqs & below);
        if (gt || (eq && e < left)) kept[L + __popc(gts & below) + min(e, left)] = run + 32 * step + lane;
        L += __popc(gts);
        E += __popc(eqs);
    });
}

// A thread per 16-byte chunk of U kept entries at a time (position, page and chunk
// are loads that wait for one another, so several chains run side by side);
// then the weights, with zeros behind the kept ones.  Bound by its bytes: 16 x 8192
// entries of 8 heads of 128 in f16, 135 MB, 26 us (5.2 TB/s).
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
            s[u] += s[u] < 0 ? 0 : (int64_t)(x - j * cpr) * 16;
            d[u] += d[u] < 0 ? 0 : (int64_t)(x - j * cpr) * 16;
        }
        // an entry whose page is not in the pool is NaN (of every type), as it was, and
        // not what the new page holds
#pragma unroll
        for (int u = 0; u < U; u++) {
            k[u] = v[u] = make_uint4(LOST, LOST, LOST, LOST);
            if (s[u] >= 0 && d[u] >= 0) {
                k[u] = *(const uint4 *)(kb + s[u]);
                v[u] = *(const uint4 *)(vb + s[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (d[u] >= 0) {
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

// Blocks of a cluster: enough that a thread has at most 16 of the weights a row may
// have, 8 at most.  Clusters of up to 16 against 8, rows and heads of 131072 weights,
// with the copy of the weights: one 15.8 / 18.3 us, 16 39 / 33, 64 112 / 80: they wait
// for one another's place.
int launch_select(const EvictArgs &a, unsigned rows, cudaStream_t st) {
    int size = 1;
    while (size < MOST && size * SEL * 16 < a.width) size <<= 1;
    const int most = (a.width + size * SEL - 1) / (size * SEL), held = most < HELD ? most : HELD;
    FOCR_CUDA_TRY(set_max_dynamic_smem((const void *)evict_select_kernel, HELD * SEL * 4));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size, a.c.kv_heads, rows);
    cfg.blockDim = SEL;
    cfg.dynamicSmemBytes = (size_t)held * SEL * 4;
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

extern "C" int focr_paged_evict(const focr_paged_cache *cache, const focr_paged_evict_args *args, void *stream) {
    return guarded("paged_evict", [&]() -> int {
        if (!args) return fail(FOCR_E_ARG, "paged_evict: null arguments");
        const int32_t *lens = args->lens;
        const float *weights = args->weights;
        const int32_t *new_table = args->new_table;
        int32_t *kept = args->kept;
        int32_t *lens_out = args->lens_out;
        float *weights_out = args->weights_out;
        const size_t rows = args->rows;
        const size_t width = args->width;
        const size_t weights_row_stride = args->weights_row_stride;
        const size_t weights_head_stride = args->weights_head_stride;
        const size_t new_table_stride = args->new_table_stride;
        const size_t new_pages = args->new_pages;
        const size_t budget = args->budget;
        const size_t sink = args->sink;
        const size_t recent = args->recent;
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
        a.width = (int)width;
        a.budget = (int)budget;
        a.sink = (int)sink;
        a.recent = (int)recent;
        cudaStream_t st = (cudaStream_t)stream;
        if ((rc = launch_select(a, (unsigned)rows, st))) return rc;
        const size_t n = budget * (a.c.row_bytes / 16), most = n > width ? n : width;
        const unsigned blocks = (unsigned)((most + 1023) / 1024);
        FOCR_CUDA_TRY(launch_pdl(evict_gather_kernel, dim3(blocks < 256 ? blocks : 256, cache->kv_heads, (unsigned)rows),
                                 256, 0, st, a));
        return FOCR_OK;
    });
}
