// Attention of one new token per row over a paged K/V cache.
//
//   s_j = scale * q . k_j          over the row's visible positions j
//   p   = softmax(s),  out = sum_j p_j v_j,  weights[j] += sum over the
//   query heads of j's kv head of p_j
//
// A position j of a row of length n is visible when j < n and (no window, or
// j < ref, or j >= n - window).  The visible positions are numbered 0..vis-1
// without the gap, so hidden ones cost nothing.
//
// One pass over K and V with a running maximum and sum (base-2 exponentials
// of c * s, c = scale * log2 e); partial results join by
//   M = max m_i,  L = sum l_i 2^(c m_i - c M),  out = sum a_i 2^(c m_i - c M) / L.
// Everything is held in f32; only K/V themselves have the cache's type, and
// the output is rounded once to q's type.
//
// Work split: the lengths are on the device, so the host cannot lay out the
// split.  The unit is a block tile (4 warp tiles of KEYS positions); all units
// of all (row, head)s are numbered in order and every block of a fixed grid
// takes an equal run of them, wherever rows begin and end.  A block that covers
// a (row, head) whole writes the output; pieces go to the workspace (a block
// has at most two) and paged_join_kernel joins them.  So no row length, however
// ragged the batch, leaves SMs idle.
//
// Short rows wait on latency, not on bytes.  There a block, or a cluster of blocks,
// has each (row, head) to itself and joins its pieces through distributed shared
// memory, which saves the second kernel; and where there are many of a few tiles, a
// warp has each and joins nothing.
#pragma once

#include <cooperative_groups.h>

#include <type_traits>

#include "paged.cuh"

namespace focr {

namespace cg = cooperative_groups;

constexpr int ATTN_WARPS = 4, ATTN_ROWS = 1024;  // rows of one launch
constexpr int ATTN_HEADS = 16;                   // most query heads a block takes together

// Rows of one launch behind a table of `cap` positions: their tiles, of 32 positions or
// more, are counted in 32 bits, however many rows share the pages.
constexpr int attn_rows(size_t cap) {
    const size_t tiles = (cap + 31) / 32, fit = tiles ? INT32_MAX / tiles : ATTN_ROWS;
    return fit < ATTN_ROWS ? (int)fit : ATTN_ROWS;
}
static_assert(attn_rows(0) == ATTN_ROWS && attn_rows(1u << 25) == ATTN_ROWS && attn_rows(1u << 26) == ATTN_ROWS - 1 &&
              attn_rows((size_t)INT32_MAX - 65535) == 32, "at least one row, at most 2^31 - 1 tiles");

// How the work is shared out, where not by clusters: runs of block tiles, or a (row,
// head) for each warp.
constexpr int RUNS = 0, SOLO = -1;

struct AttnArgs {
    PagedView c;
    const void *q;
    const int32_t *lens, *refs;
    void *out;
    float *scores;   // raw s of every (row, q head, visible index), only when weights are asked for
    float2 *stat;    // (M, 1 / L) of every (row, q head), likewise
    float *part;     // [block][2][gp][dim] partial sums
    float2 *ml;      // [block][2][gp] partial (m, l)
    long long q_stride, out_stride;
    int rows, group, q_heads, dim, q_type, window, cap, width;
    int score_stride;     // floats between the scores of two query heads, even
    int gp, head_chunks;  // query heads that a block takes together; blocks of them a kv head
    int tile_shift;       // log2 of a block tile's positions
    int cluster;          // blocks that share one (row, head); RUNS or SOLO
    float c2;             // scale * log2(e)
};

// The visible positions of row r: index i is position i below `ref` and
// i + gap from there on.  bad: the row's length passes its table or weights.
struct RowView {
    int vis, ref, gap;
    bool bad;
};
__device__ __forceinline__ RowView row_view(const AttnArgs &a, int r) {
    RowView v{0, 0, 0, false};
    const int n = a.lens[r];
    if (n <= 0) return v;
    if (n > a.cap) {
        v.bad = true;
        return v;
    }
    v.ref = v.vis = n;
    if (a.window > 0) {
        int ref = a.refs ? a.refs[r] : 0;
        ref = ref < 0 ? 0 : ref > n ? n : ref;
        const int start = max(ref, n - min(a.window, n));
        v.ref = ref;
        v.gap = start - ref;
        v.vis = n - v.gap;
    }
    return v;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The maximum that scores are taken relative to: 0 where all are -inf.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
// 2^(c (s - m)), m from base_of.  The difference comes first: a product of m and c of its
// own would be rounded by more than the exponential bears where it passes 2^24, as the
// lowest finite values in all of a row's keys make it.
__device__ __forceinline__ float prob(float s, float c, float m) { return ex2(__fmul_rn(__fsub_rn(s, m), c)); }
// What takes sums relative to the maximum m over to the maximum top >= m; exactly 1 where
// the maximum stays.
__device__ __forceinline__ float rescale(float m, float top, float c) { return m == -INFINITY ? 0.0f : prob(m, c, top); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Prefix of the rows' tile counts into `pre` (ATTN_ROWS + 1 ints), by a block of
// NT threads.
template <int NT> __device__ void tile_prefix(const AttnArgs &a, int *pre) {
    constexpr int PER = ATTN_ROWS / NT;
    __shared__ int wsum[NT / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int round = (1 << a.tile_shift) - 1;
    if (a.rows <= 32) {  // one warp's scan; the usual small batch
        if (warp == 0) {
            int inc = lane < a.rows ? (row_view(a, lane).vis + round) >> a.tile_shift : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            if (lane < a.rows) pre[lane + 1] = inc;
            if (lane == 0) pre[0] = 0;
        }
        __syncthreads();
        return;
    }
    int n[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = t * PER + i;
        n[i] = r < a.rows ? (row_view(a, r).vis + round) >> a.tile_shift : 0;
        sum += n[i];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < warp; w++) before += wsum[w];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = t * PER + i;
        if (r <= a.rows) pre[r] = before;
        before += n[i];
    }
    if (t == NT - 1 && a.rows == ATTN_ROWS) pre[ATTN_ROWS] = before;
    __syncthreads();
}

// Blocks that get units: every one of them gets at least one.
__device__ __forceinline__ unsigned long long run_count(unsigned long long total, int blocks) {
    return min(total, (unsigned long long)blocks);
}

// The last row whose units begin at or before u.
__device__ __forceinline__ int row_of_unit(const int *pre, int rows, int hc_count, unsigned long long u) {
    int lo = 0, hi = rows;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((unsigned long long)pre[mid] * hc_count <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The run of units of one block, and the piece of a (row, kv head, chunk of its
// query heads) it stands at.
struct Segment {
    int r, kvh, heads, qh0, t0, t1;
    int slot;      // of a piece, in runs
    bool whole;
    RowView rv;
};
// n / d; most calls fit 32 bits, whose division is several times shorter.
__device__ __forceinline__ unsigned long long quotient(unsigned long long n, unsigned long long d) {
    return (n | d) >> 32 ? n / d : (uint32_t)n / (uint32_t)d;
}

template <bool ALONE> struct Run {
    unsigned long long left;     // units to come
    int r, kvh, chunk, t, tiles; // where the next one lies: tile t of `tiles`
    int unit;                    // the next (row, head), counted, of a warp of its own
    bool first;

    // The run of this block; in a cluster its share of the cluster's (row, head),
    // which may be empty.
    __device__ Run(const AttnArgs &a, const int *pre) {
        if constexpr (ALONE) {
            unit = blockIdx.x * ATTN_WARPS + (threadIdx.x >> 5);
            return;
        }
        if (a.cluster) {
            const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
            const int row_units = a.c.kv_heads * a.head_chunks;
            r = unit / row_units;
            kvh = (unit - r * row_units) / a.head_chunks;
            chunk = unit - r * row_units - kvh * a.head_chunks;
            const int n = (row_view(a, r).vis + (1 << a.tile_shift) - 1) >> a.tile_shift;
            const int per = n / a.cluster, rest = n - per * a.cluster;   // the first `rest` blocks have one more
            t = rank * per + min(rank, rest);
            tiles = t + per + (rank < rest);
            left = tiles - t;
            first = true;
            return;
        }
        const int hc_count = a.c.kv_heads * a.head_chunks;
        const unsigned long long total = (unsigned long long)pre[a.rows] * hc_count;
        const unsigned long long runs = run_count(total, gridDim.x);
        left = 0;
        if (blockIdx.x >= runs) return;
        const unsigned long long u = quotient(blockIdx.x * total, runs);
        left = quotient((blockIdx.x + 1ull) * total, runs) - u;
        r = row_of_unit(pre, a.rows, hc_count, u);
        tiles = pre[r + 1] - pre[r];
        const unsigned long long off = u - (unsigned long long)pre[r] * hc_count;
        const int hc = (int)quotient(off, tiles);
        t = (int)(off - (unsigned long long)hc * tiles);
        kvh = hc / a.head_chunks;
        chunk = hc - kvh * a.head_chunks;
        first = true;
    }
    __device__ bool next(const AttnArgs &a, const int *pre, Segment *s) {
        if constexpr (ALONE) {
            const int per_row = a.c.kv_heads * a.head_chunks;
            r = unit / per_row;
            if (r >= a.rows) return false;
            kvh = (unit - r * per_row) / a.head_chunks;
            chunk = unit - r * per_row - kvh * a.head_chunks;
            unit += gridDim.x * ATTN_WARPS;
            s->rv = row_view(a, r);
            s->t0 = 0;
            s->t1 = (s->rv.vis + (1 << a.tile_shift) - 1) >> a.tile_shift;
            s->r = r;
            s->kvh = kvh;
            s->heads = min(a.gp, a.group - chunk * a.gp);
            s->qh0 = kvh * a.group + chunk * a.gp;
            return true;
        }
        // a cluster's blocks all take part in its join
        if (a.cluster ? !first : !left) return false;
        if (t == tiles && !a.cluster) {   // the next (row, kv head, chunk)
            t = 0;
            if (++chunk == a.head_chunks) {
                chunk = 0;
                if (++kvh == a.c.kv_heads) {
                    kvh = 0;
                    do {
                        r++;
                        tiles = pre[r + 1] - pre[r];
                    } while (tiles == 0);   // units are left: a row with some follows
                }
            }
        }
        s->r = r;
        s->t0 = t;
        s->t1 = (int)min((unsigned long long)tiles, t + left);
        s->whole = t == 0 && s->t1 == tiles;
        s->slot = blockIdx.x * 2 + (first ? 0 : 1);
        s->kvh = kvh;
        s->heads = min(a.gp, a.group - chunk * a.gp);
        s->qh0 = kvh * a.group + chunk * a.gp;
        s->rv = row_view(a, r);
        left -= s->t1 - t;
        t = s->t1;
        first = false;
        return true;
    }
};

// The first position of a warp's part of a tile.
template <int KEYS, bool ALONE> __device__ __forceinline__ int first_key(int tile, int warp) {
    return (ALONE ? tile : tile * ATTN_WARPS + warp) * KEYS;
}

// The tiles of a block's run in order, across its segments, for the copies that run
// ahead of the arithmetic.  A warp's lane `i` finds the place of the tile's i-th
// position.
template <int KEYS, bool ALONE> struct Feed {
    Run<ALONE> run;
    const int32_t *pages;
    int64_t head;          // the kv head's offset in a page
    RowView rv;
    int tile, end;

    __device__ explicit Feed(const Run<ALONE> &r) : run(r), tile(0), end(0) {}
    // The byte offset of this lane's position of the next tile, -1 where there is
    // none; *bad if its page is not in the pool.
    __device__ int64_t next(const AttnArgs &a, const int *pre, int warp, int lane, bool *bad) {
        *bad = false;
        while (tile == end) {   // a row of a warp's own may have no tiles
            Segment s;
            if (!run.next(a, pre, &s)) return -1;
            pages = a.c.table + s.r * a.c.table_stride;
            head = s.kvh * a.c.head_stride;
            rv = s.rv;
            tile = s.t0;
            end = s.t1;
        }
        const int i = first_key<KEYS, ALONE>(tile++, warp) + lane;
        if (lane >= KEYS || i >= rv.vis) return -1;
        const int64_t o = a.c.offset(pages, (uint32_t)(i < rv.ref ? i : i + rv.gap));
        *bad = o < 0;
        return o < 0 ? o : o + head;
    }
};

// Four neighbouring elements, as one store where they lie on its boundary.
__device__ __forceinline__ void store4_as(void *p, int dtype, int64_t i, float4 x) {
    if (dtype == FOCR_F32) {
        float *q = static_cast<float *>(p) + i;
        if ((uintptr_t)q % 16 == 0) {
            *reinterpret_cast<float4 *>(q) = x;
            return;
        }
    } else {
        uint16_t *q = static_cast<uint16_t *>(p) + i;
        if ((uintptr_t)q % 8 == 0) {
            alignas(8) uint16_t y[4];
            store_f32_as(y, dtype, 0, x.x);
            store_f32_as(y, dtype, 1, x.y);
            store_f32_as(y, dtype, 2, x.z);
            store_f32_as(y, dtype, 3, x.w);
            *reinterpret_cast<uint2 *>(q) = *reinterpret_cast<const uint2 *>(y);
            return;
        }
    }
    store_f32_as(p, dtype, i, x.x);
    store_f32_as(p, dtype, i + 1, x.y);
    store_f32_as(p, dtype, i + 2, x.z);
    store_f32_as(p, dtype, i + 3, x.w);
}
// Two of them.
__device__ __forceinline__ void store2_as(void *p, int dtype, int64_t i, float x, float y) {
    if (dtype == FOCR_F32) {
        float *q = static_cast<float *>(p) + i;
        if ((uintptr_t)q % 8 == 0) {
            *reinterpret_cast<float2 *>(q) = make_float2(x, y);
            return;
        }
    } else {
        uint16_t *q = static_cast<uint16_t *>(p) + i;
        if ((uintptr_t)q % 4 == 0) {
            alignas(4) uint16_t z[2];
            store_f32_as(z, dtype, 0, x);
            store_f32_as(z, dtype, 1, y);
            *reinterpret_cast<uint32_t *>(q) = *reinterpret_cast<const uint32_t *>(z);
            return;
        }
    }
    store_f32_as(p, dtype, i, x);
    store_f32_as(p, dtype, i + 1, y);
}
__device__ __forceinline__ float4 fma4(float4 x, float f, float4 o) {
    return make_float4(__fmaf_rn(x.x, f, o.x), __fmaf_rn(x.y, f, o.y), __fmaf_rn(x.z, f, o.z),
                       __fmaf_rn(x.w, f, o.w));
}
// x / L; 0 where the row sees nothing, of whose sums L is 0 or, for a bad length, NaN.
// Where it does see something, but all with scores of -inf, L is 0 too and 0 / 0 is right.
__device__ __forceinline__ float4 over4(float4 x, float L, bool sees) {
    if (!sees && L == 0.0f) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(x.x / L, x.y / L, x.z / L, x.w / L);
}

// What the warps of a block hand over at the end of a segment: HR heads at a time,
// beside the rings, into which the next segment's rows are already flowing.  A
// cluster's blocks then hand their joined part to one another in the first warp's
// place.
template <int HR, int D> struct Handover {
    float o[ATTN_WARPS][HR][D], m[ATTN_WARPS][HR], l[ATTN_WARPS][HR];
};

// Joins the block's warps for the heads g0 .. g0 + HR - 1 of the segment, and
// writes their output or piece.  The block waits for it at the end.
template <int GP, int HR, int D>
__device__ __forceinline__ void finish_heads(const AttnArgs &a, const Segment &s, Handover<HR, D> &h, int g0) {
    const int n = min(HR, s.heads - g0) * (D / 4);
    for (int x = threadIdx.x; x < n; x += ATTN_WARPS * 32) {
        const int i = x / (D / 4), g = g0 + i, d = x % (D / 4) * 4;
        if (d >= a.dim) continue;   // a multiple of 4
        float M = -INFINITY, L = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < ATTN_WARPS; w++) M = fmaxf(M, h.m[w][i]);
#pragma unroll
        for (int w = 0; w < ATTN_WARPS; w++) {
            const float f = rescale(h.m[w][i], M, a.c2);
            L = __fmaf_rn(h.l[w][i], f, L);
            o = fma4(*reinterpret_cast<const float4 *>(&h.o[w][i][d]), f, o);
        }
        if (a.cluster > 1) {
            // only this thread reads these four; the other threads still read m and l
            *reinterpret_cast<float4 *>(&h.o[0][i][d]) = o;
            if (d == 0) {
                h.o[1][i][0] = M;
                h.o[1][i][1] = L;
            }
        } else if (s.whole) {
            store4_as(a.out, a.q_type, s.r * a.out_stride + (long long)(s.qh0 + g) * a.dim + d, over4(o, L, s.rv.vis));
            if (a.stat && d == 0) a.stat[(int64_t)s.r * a.q_heads + s.qh0 + g] = make_float2(M, 1.0f / L);
        } else {
            *reinterpret_cast<float4 *>(a.part + ((int64_t)s.slot * GP + g) * a.dim + d) = o;
            if (d == 0) a.ml[s.slot * GP + g] = make_float2(M, L);
        }
    }
    if (a.cluster <= 1) {
        __syncthreads();
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int x = cluster.block_rank() * (ATTN_WARPS * 32) + threadIdx.x; x < n; x += a.cluster * (ATTN_WARPS * 32)) {
        const int i = x / (D / 4), g = g0 + i, d = x % (D / 4) * 4;
        if (d >= a.dim) continue;
        float M = -INFINITY, L = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int q = 0; q < a.cluster; q++) M = fmaxf(M, cluster.map_shared_rank(&h, q)->o[1][i][0]);
#pragma unroll 8
        for (int q = 0; q < a.cluster; q++) {
            const Handover<HR, D> *y = cluster.map_shared_rank(&h, q);
            const float2 ml = *reinterpret_cast<const float2 *>(&y->o[1][i][0]);
            const float f = rescale(ml.x, M, a.c2);
            L = __fmaf_rn(ml.y, f, L);
            o = fma4(*reinterpret_cast<const float4 *>(&y->o[0][i][d]), f, o);
        }
        store4_as(a.out, a.q_type, s.r * a.out_stride + (long long)(s.qh0 + g) * a.dim + d, over4(o, L, s.rv.vis));
        if (a.stat && d == 0) a.stat[(int64_t)s.r * a.q_heads + s.qh0 + g] = make_float2(M, 1.0f / L);
    }
    cluster.sync();   // nobody overwrites or leaves what another still reads
}

// The rows that have no units, shared out over the blocks: zeros where nothing is
// visible, NaN for a length that passes the table.
__device__ __forceinline__ void finish_empty_rows(const AttnArgs &a, const int *pre) {
    if (a.cluster != RUNS) return;   // elsewhere a row has a segment, if an empty one
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        if (pre[r + 1] != pre[r]) continue;
        const float x = row_view(a, r).bad ? NAN : 0.0f;
        for (int i = threadIdx.x; i < a.q_heads * a.dim; i += ATTN_WARPS * 32)
            store_f32_as(a.out, a.q_type, r * a.out_stride + i, x);
    }
}

inline int ilog2(int x) {
    int n = 0;
    while ((1 << n) < x) n++;
    return n;
}
inline int attn_blocks() { return num_sms() * 2; }

// Launches an attention kernel as a.cluster says.
template <typename K> int launch_attn(K kernel, int smem, const AttnArgs &a, cudaStream_t st) {
    FOCR_CUDA_TRY(set_max_dynamic_smem((const void *)kernel, smem));
    if (a.cluster <= 0) {
        const size_t units = (size_t)a.rows * a.c.kv_heads * a.head_chunks, warps = (size_t)attn_blocks() * ATTN_WARPS;
        const int blocks = a.cluster == SOLO && units < warps ? (int)((units + ATTN_WARPS - 1) / ATTN_WARPS) : attn_blocks();
        FOCR_CUDA_TRY(launch_pdl(kernel, blocks, ATTN_WARPS * 32, smem, st, a));
        return FOCR_OK;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = a.rows * a.c.kv_heads * a.head_chunks * a.cluster;
    cfg.blockDim = ATTN_WARPS * 32;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    FOCR_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
    return FOCR_OK;
}

// How a call is shared out.  The visible positions of a row are not known here, only
// its table's capacity.
// A cluster saves the prefix, the cuts and the join, and the hardware hands out the
// rows; runs are even however long one row is.  So: as many blocks as fit the SMs at two
// each (at head_dim 256 the tensor cores' blocks, and those of an f32 cache, fit one an
// SM: there the split was not measured apart), 8 at most, where each has at most 128 KB
// of K to read, 256 KB where most SMs are busy, twice that where 16 heads would be handed
// over in pieces; and one block a (row, head) for up to four times as many as fit.
// Clusters against runs:
//   1 row, 10 heads of f32: 1024 positions 7.7 / 10.5 us, 2048 10.4 / 11.7, 4096 (256 KB
//   on a quarter of the SMs, not taken) 15.4 / 13.6;
//   8 rows x 8 heads of bf16: 256 positions 7.2 / 9.7, 2048 14.0 / 17.3; 32 x 8: 64 5.6 /
//   7.6, 512 12.5 / 17.2, 1024 (256 KB) 25.7 / 30.6; 512 in one row, the others short:
//   10.4 / 11.4;
//   19 x 5 with 8 query heads: 1536 23.3 / 24.5, ragged 21.3 / 24.9, one long 19.7 / 17.1;
//   80 of f32, 1024 positions: 3 blocks 15.0, 2 18.5, runs 18.3;
//   64 x 10 of 1 to 512 positions 22.9 / 29.1, of 512 each 39.0 / 37.4; 4 query heads 31.9
//   / 44.0 and 47.5 / 42.5; 256 x 16 of 128 each (not taken) 84 / 64.
// Where there are more (row, head)s than blocks fit, a warp takes one: nothing is joined
// or waited for, but its tiles, about 0.9 us each, follow one another.  Up to a
// fortieth of the (row, head)s, 48 at most, the longest row ends about when the others
// do.  bf16, full tables, warps against the better of the above, for one query head and
// for four: 40 x 8: 64 positions (4 tiles) 7.0 / 9.2 us and 10.4 / 13.3, 128 9.7 / 11.0
// and 13.5 / 15.1, 256 (16 tiles, not taken) 15.1 / 14.7 and 19.6 / 19.6, ragged 14.7 /
// 10.9 and 19.2 / 15.2; 128 x 8: 16 5.4 / 14.6 and 8.8 / 21.0, 256 25.7 / 33.9 and 28.8 /
// 40.9; 224 x 16: 16 13.5 / 34.5 and 26.2 / 54.4, 128 47.5 / 58.2 and 59.4 / 74.8, 512 (32
// tiles) 152 / 148 and 168 / 164, ragged 88.4 / 103.5 and 101.8 / 140.1.  `keys`: of a
// warp's tile, 0 where the kernel's warps cannot work alone.
inline int cluster_of(const AttnArgs &a, int keys) {
    const size_t units = (size_t)a.rows * a.c.kv_heads * a.head_chunks, most = (size_t)attn_blocks();
    const size_t tiles = keys ? ((size_t)a.cap + keys - 1) / keys : SIZE_MAX;
    if (units > most && tiles <= 48 && tiles * 40 <= units) return SOLO;
    size_t n = 8;   // clusters of 5 and more leave gaps between them, those of 2 none
    while (n > 1 && units * n * 16 > most * (n > 4 ? 13 : n > 2 ? 14 : 16)) n--;
    const size_t bytes = (size_t)a.cap * a.c.row_bytes;
    const int shift = (units * n * 4 >= most * 3 ? 18 : 17) + (a.gp == 16);
    if (units > most * 4 || bytes > n << shift) return RUNS;
    return (int)n;
}

// The attention kernel for one type of cache, without the join; sets gp,
// head_chunks and tile_shift of `a` as that kernel has them.
int launch_attention_f32(AttnArgs &a, cudaStream_t st);
int launch_attention_f16(AttnArgs &a, cudaStream_t st);
int launch_attention_bf16(AttnArgs &a, cudaStream_t st);

}  // namespace focr
