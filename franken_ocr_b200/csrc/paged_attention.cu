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
//   M = max m_i,  L = sum l_i 2^(c (m_i - M)),  out = sum a_i 2^(c (m_i - M)) / L.
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
#include <type_traits>

#include "paged.cuh"

namespace focr {
namespace {

constexpr int WARPS = 4, MAX_ROWS = 1024;

struct AttnArgs {
    PagedView c;
    const void *q;
    const int32_t *lens, *refs;
    void *out;
    float *scores;   // raw s of every (row, q head, visible index), only when weights are asked for
    float2 *stat;    // (M, 1 / L) of every (row, q head), likewise
    float *part;     // [block][2][GP][dim] partial sums
    float2 *ml;      // [block][2][GP] partial (m, l)
    long long q_stride, out_stride;
    int rows, group, head_chunks, q_heads, dim, q_type, window, cap, width;
    float c2;        // scale * log2(e)
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
// 2^(c (s - m)) with m's product rounded once, the same for every s of a row.
__device__ __forceinline__ float prob(float s, float c, float mc) { return ex2(__fmaf_rn(s, c, -mc)); }
__device__ __forceinline__ float scaled_max(float m, float c) {
    return m == -INFINITY ? 0.0f : __fmul_rn(m, c);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Prefix of the rows' tile counts into `pre` (MAX_ROWS + 1 ints), by a block of
// WARPS * 32 threads.
template <int TILE> __device__ void tile_prefix(const AttnArgs &a, int *pre) {
    constexpr int PER = MAX_ROWS / (WARPS * 32);
    __shared__ int wsum[WARPS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    int n[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = t * PER + i;
        n[i] = r < a.rows ? (row_view(a, r).vis + TILE - 1) / TILE : 0;
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
    if (t == WARPS * 32 - 1 && a.rows == MAX_ROWS) pre[MAX_ROWS] = before;
    __syncthreads();
}

// Blocks that get units: every one of them gets at least one.
__device__ __forceinline__ unsigned long long run_count(unsigned long long total, int blocks) {
    return min(total, (unsigned long long)blocks);
}

// Shapes of a warp tile.  A row of D elements is DB bytes; LPK lanes share a
// key (NC 16-byte chunks each), KPI keys go by per step, ITS steps a tile.
template <typename T, int D> struct Tile {
    static constexpr int DB = D * (int)sizeof(T);
    static constexpr int LPK = DB / 16 < 32 ? DB / 16 : 32;
    static constexpr int NC = DB / 16 / LPK;
    static constexpr int KPI = 32 / LPK;
    static constexpr int ITS = 8;
    static constexpr int KEYS = ITS * KPI;
    static constexpr int HALF = KEYS * DB;      // bytes of K, and of V, in a stage
    static constexpr int STAGES = HALF > 4096 ? 2 : 3;
    static constexpr int BLOCK = WARPS * KEYS;  // positions of a block tile
    static constexpr int EPL = NC * 16 / (int)sizeof(T);  // dimensions of a lane
};

template <typename T, int D, int GP> constexpr int attn_smem() {
    using S = Tile<T, D>;
    return WARPS * S::STAGES * 2 * S::HALF + WARPS * GP * S::KEYS * 4 + (MAX_ROWS + 1) * 4;
}

// The arithmetic runs on the f32 units: with few query heads a kv head the
// loads bound it (a key of 128 16-bit values costs a warp ~25 instructions a
// head against 512 bytes).
template <typename T, int D, int GP>
__global__ void __launch_bounds__(WARPS * 32, 2) paged_attention_kernel(const AttnArgs a) {
    using S = Tile<T, D>;
    constexpr int LPK = S::LPK, KPI = S::KPI, ITS = S::ITS, KEYS = S::KEYS, NC = S::NC, EPL = S::EPL;
    constexpr int EPC = 16 / (int)sizeof(T);  // elements of a chunk
    extern __shared__ __align__(128) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    char *ring = smem + warp * S::STAGES * 2 * S::HALF;
    float *probs = reinterpret_cast<float *>(smem + WARPS * S::STAGES * 2 * S::HALF) + warp * GP * KEYS;
    int *pre = reinterpret_cast<int *>(smem + WARPS * S::STAGES * 2 * S::HALF + WARPS * GP * KEYS * 4);
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);

    pdl_wait();
    pdl_trigger();
    tile_prefix<S::BLOCK>(a, pre);
    const int HC = a.c.kv_heads * a.head_chunks;
    const unsigned long long total = (unsigned long long)pre[a.rows] * HC;
    const unsigned long long runs = run_count(total, gridDim.x);
    if (blockIdx.x >= runs) return;
    unsigned long long u = blockIdx.x * total / runs;
    const unsigned long long u_begin = u, u_end = (blockIdx.x + 1ull) * total / runs;

    const int sub = lane / LPK, chunk = lane % LPK;
    // the step whose score this lane holds after the transposing reduction
    const int my_it = (lane & (LPK / 2) ? 4 : 0) + (lane & (LPK / 4) ? 2 : 0) + (lane & (LPK / 8) ? 1 : 0);
    const int my_key = my_it * KPI + sub;

    while (u < u_end) {
        // the (row, head) of unit u: the last row whose units begin at or before u
        int lo = 0, hi = a.rows;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((unsigned long long)pre[mid] * HC <= u) lo = mid;
            else hi = mid;
        }
        const int r = lo;
        const int tiles = pre[r + 1] - pre[r];
        const unsigned long long off = u - (unsigned long long)pre[r] * HC;
        const int hc = (int)(off / tiles), t0 = (int)(off - (unsigned long long)hc * tiles);
        const int t1 = (int)min((unsigned long long)tiles, t0 + (u_end - u));
        const bool at_start = u == u_begin;
        u += t1 - t0;

        const RowView rv = row_view(a, r);
        const int kvh = hc / a.head_chunks, g0 = (hc - kvh * a.head_chunks) * GP;
        const int heads = min(GP, a.group - g0), qh0 = kvh * a.group + g0;
        const int32_t *pages = a.c.table + r * a.c.table_stride;
        const char *kb = a.c.k + kvh * a.c.head_stride, *vb = a.c.v + kvh * a.c.head_stride;

        float q[GP][EPL], acc[GP][EPL], m[GP], l[GP];
#pragma unroll
        for (int g = 0; g < GP; g++) {
            m[g] = -INFINITY;
            l[g] = 0.0f;
#pragma unroll
            for (int e = 0; e < EPL; e++) {
                const int d = (e / EPC * LPK + chunk) * EPC + e % EPC;
                q[g][e] = g < heads && d < a.dim
                              ? load_as_f32(a.q, a.q_type, r * a.q_stride + (long long)(qh0 + g) * a.dim + d)
                              : 0.0f;
                acc[g][e] = 0.0f;
            }
        }
        bool bad = false;

        auto key_offset = [&](int tile) -> int64_t {  // of index `lane` of the warp's tile
            const int i = (tile * WARPS + warp) * KEYS + lane;
            if (lane >= KEYS || i >= rv.vis || tile >= t1) return -1;
            const int64_t o = a.c.offset(pages, (uint32_t)(i < rv.ref ? i : i + rv.gap));
            bad |= o < 0;
            return o;
        };
        auto issue = [&](int stage, int64_t mine) {
            const uint32_t dst = ring_s + stage * 2 * S::HALF + lane * 16;
#pragma unroll
            for (int it = 0; it < ITS; it++) {
                const int64_t o = __shfl_sync(0xffffffffu, mine, it * KPI + sub);
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    const int b = (n * LPK + chunk) * 16;
                    const bool have = o >= 0 && b < a.c.row_bytes;
                    const int64_t src = have ? o + b : 0;
                    cp_async16(dst + (it * NC + n) * 512, kb + src, have ? 16 : 0);
                    cp_async16(dst + S::HALF + (it * NC + n) * 512, vb + src, have ? 16 : 0);
                }
            }
        };
#pragma unroll
        for (int s = 0; s < S::STAGES; s++) {
            issue(s, key_offset(t0 + s));
            cp_async_commit();
        }
        int stage = 0;
        for (int tile = t0; tile < t1; tile++) {
            const int64_t next = key_offset(tile + S::STAGES);
            cp_async_wait<S::STAGES - 1>();
            __syncwarp();
            const char *ks = ring + stage * 2 * S::HALF + lane * 16, *vs = ks + S::HALF;
            // scores: partial dots of every step, then each lane's own key
            float s[GP][ITS];
#pragma unroll
            for (int it = 0; it < ITS; it++) {
                float kf[EPL];
#pragma unroll
                for (int n = 0; n < NC; n++)
                    unpack16<T>(*reinterpret_cast<const uint4 *>(ks + (it * NC + n) * 512), kf + n * EPC);
#pragma unroll
                for (int g = 0; g < GP; g++) {
                    float d = 0.0f;
#pragma unroll
                    for (int e = 0; e < EPL; e++) d = __fmaf_rn(q[g][e], kf[e], d);
                    s[g][it] = d;
                }
            }
            const int i = (tile * WARPS + warp) * KEYS + my_key;
            const bool live = i < rv.vis;
#pragma unroll
            for (int g = 0; g < GP; g++) {
                // transposing reduction: 8 values over LPK lanes leave one a lane
#pragma unroll
                for (int half = 4; half > 0; half >>= 1) {
                    const int o = LPK * half / 8;
                    const bool up = lane & o;
#pragma unroll
                    for (int x = 0; x < half; x++) {
                        const float give = up ? s[g][x] : s[g][x + half];
                        const float keep = up ? s[g][x + half] : s[g][x];
                        s[g][x] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
                }
#pragma unroll
                for (int o = LPK / 16; o > 0; o >>= 1) s[g][0] += __shfl_xor_sync(0xffffffffu, s[g][0], o);
                const float sc = live ? s[g][0] : -INFINITY;
                if (__any_sync(0xffffffffu, sc > m[g])) {
                    const float top = fmaxf(m[g], warp_max_f32(sc));
                    const float f = prob(m[g], a.c2, scaled_max(top, a.c2));
                    m[g] = top;
                    l[g] *= f;
#pragma unroll
                    for (int e = 0; e < EPL; e++) acc[g][e] *= f;
                }
                const float p = prob(sc, a.c2, scaled_max(m[g], a.c2));
                l[g] += p;
                probs[g * KEYS + sub * ITS + my_it] = p;
                if (a.scores && live && g < heads)
                    a.scores[((int64_t)r * a.q_heads + qh0 + g) * a.width + i] = sc;
            }
            __syncwarp();
#pragma unroll
            for (int it = 0; it < ITS; it++) {
                float vf[EPL];
#pragma unroll
                for (int n = 0; n < NC; n++)
                    unpack16<T>(*reinterpret_cast<const uint4 *>(vs + (it * NC + n) * 512), vf + n * EPC);
#pragma unroll
                for (int g = 0; g < GP; g++) {
                    const float p = probs[g * KEYS + sub * ITS + it];
#pragma unroll
                    for (int e = 0; e < EPL; e++) acc[g][e] = __fmaf_rn(p, vf[e], acc[g][e]);
                }
            }
            __syncwarp();
            issue(stage, next);
            cp_async_commit();
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        }
        cp_async_wait<0>();

        // the warp's sums over its lanes, then the block's over its warps,
        // through the rings (no copy is in flight)
        const bool any_bad = __any_sync(0xffffffffu, bad);
        __syncwarp();
        float *mine = reinterpret_cast<float *>(ring);  // [GP][D], then m[GP], l[GP]
#pragma unroll
        for (int g = 0; g < GP; g++) {
            float lsum = l[g];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, o);
            lsum *= 8.0f / LPK;  // LPK / 8 lanes hold the same key
#pragma unroll
            for (int e = 0; e < EPL; e++) {
                float x = acc[g][e];
#pragma unroll
                for (int o = LPK; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                if (sub == 0) mine[g * D + (e / EPC * LPK + chunk) * EPC + e % EPC] = x;
            }
            if (lane == 0) {
                mine[GP * D + g] = m[g];
                mine[GP * D + GP + g] = any_bad ? NAN : lsum;
            }
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == tiles;
        const int slot = blockIdx.x * 2 + (at_start ? 0 : 1);
        constexpr int WS = S::STAGES * 2 * S::HALF / 4;  // floats between the warps' areas
        const float *all = reinterpret_cast<const float *>(smem);
        for (int x = threadIdx.x; x < GP * D; x += WARPS * 32) {
            const int g = x / D, d = x % D;
            if (g >= heads || d >= a.dim) continue;
            float M = -INFINITY, L = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, all[w * WS + GP * D + g]);
            const float mc = scaled_max(M, a.c2);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = prob(all[w * WS + GP * D + g], a.c2, mc);
                L = __fmaf_rn(all[w * WS + GP * D + GP + g], f, L);
                o = __fmaf_rn(all[w * WS + x], f, o);
            }
            if (whole) {
                store_f32_as(a.out, a.q_type, r * a.out_stride + (long long)(qh0 + g) * a.dim + d,
                             L == 0.0f ? 0.0f : o / L);
                if (a.stat && d == 0) a.stat[(int64_t)r * a.q_heads + qh0 + g] = make_float2(M, 1.0f / L);
            } else {
                a.part[(int64_t)slot * GP * a.dim + g * a.dim + d] = o;
                if (d == 0) a.ml[slot * GP + g] = make_float2(M, L);
            }
        }
        __syncthreads();
    }
}

// Joins the pieces of one (row, kv head, chunk of its query heads) and writes
// the rows that no unit reached: zeros where nothing is visible, NaN for a
// length that passes the table.
template <int TILE, int GP>
__global__ void __launch_bounds__(WARPS * 32) paged_join_kernel(const AttnArgs a, int blocks) {
    __shared__ int pre[MAX_ROWS + 1];
    pdl_wait();
    pdl_trigger();
    tile_prefix<TILE>(a, pre);
    const int r = blockIdx.y, hc = blockIdx.x, HC = a.c.kv_heads * a.head_chunks;
    const int kvh = hc / a.head_chunks, g0 = (hc - kvh * a.head_chunks) * GP;
    const int heads = min(GP, a.group - g0), qh0 = kvh * a.group + g0;
    const int tiles = pre[r + 1] - pre[r];
    if (tiles == 0) {
        const float x = row_view(a, r).bad ? NAN : 0.0f;
        for (int i = threadIdx.x; i < heads * a.dim; i += WARPS * 32)
            store_f32_as(a.out, a.q_type, r * a.out_stride + (long long)qh0 * a.dim + i, x);
        if (a.stat && threadIdx.x < heads)
            a.stat[(int64_t)r * a.q_heads + qh0 + threadIdx.x] = make_float2(-INFINITY, NAN);
        return;
    }
    const unsigned long long total = (unsigned long long)pre[a.rows] * HC, n = run_count(total, blocks);
    const unsigned long long u0 = (unsigned long long)pre[r] * HC + (unsigned long long)hc * tiles;
    // the block whose run holds unit u: the last b with b * total / n <= u
    const int b0 = (int)(((u0 + 1) * n - 1) / total), b1 = (int)(((u0 + tiles) * n - 1) / total);
    if (b0 == b1) return;
    const int slot0 = 2 * b0 + (b0 * total / n == u0 ? 0 : 1);
    for (int x = threadIdx.x; x < heads * a.dim; x += WARPS * 32) {
        const int g = x / a.dim, d = x - g * a.dim;
        float M = -INFINITY, L = 0.0f, o = 0.0f;
        for (int b = b0; b <= b1; b++) M = fmaxf(M, a.ml[(b == b0 ? slot0 : 2 * b) * GP + g].x);
        const float mc = scaled_max(M, a.c2);
        for (int b = b0; b <= b1; b++) {
            const int s = b == b0 ? slot0 : 2 * b;
            const float2 ml = a.ml[s * GP + g];
            const float f = prob(ml.x, a.c2, mc);
            L = __fmaf_rn(ml.y, f, L);
            o = __fmaf_rn(a.part[(int64_t)s * GP * a.dim + x], f, o);
        }
        store_f32_as(a.out, a.q_type, r * a.out_stride + (long long)(qh0 + g) * a.dim + d,
                     L == 0.0f ? 0.0f : o / L);
        if (a.stat && d == 0) a.stat[(int64_t)r * a.q_heads + qh0 + g] = make_float2(M, 1.0f / L);
    }
}

// weights[r][kv head][j] += sum over the kv head's query heads of p_j, from the
// kept scores.  A row whose output is NaN leaves its weights as they were.
__global__ void __launch_bounds__(256) paged_weights_kernel(const AttnArgs a, float *weights,
                                                            long long w_row, long long w_head) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y;
    const RowView rv = row_view(a, r);
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= rv.vis) return;
    const float *s = a.scores + ((int64_t)r * a.q_heads + kvh * a.group) * a.width + i;
    const float2 *st = a.stat + (int64_t)r * a.q_heads + kvh * a.group;
    float sum = 0.0f;
    for (int g = 0; g < a.group; g++) {
        const float2 t = st[g];
        sum = __fmaf_rn(prob(s[(int64_t)g * a.width], a.c2, scaled_max(t.x, a.c2)), t.y, sum);
    }
    if (isfinite(sum)) {
        float *w = weights + r * w_row + kvh * w_head + (i < rv.ref ? i : i + rv.gap);
        *w += sum;
    }
}

// Query heads of a kv head that one block takes together.
int heads_together(int group) { return group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8; }
int attn_blocks() { return num_sms() * 2; }

struct Sizes {
    size_t scores, stat, part, ml, total;
};
Sizes attn_sizes(size_t rows, size_t q_heads, size_t dim, size_t width) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    Sizes s;
    const size_t slots = (size_t)attn_blocks() * 2 * 8;
    s.part = up(slots * dim * 4);
    s.ml = up(slots * 8);
    s.stat = width ? up(rows * q_heads * 8) : 0;
    s.scores = width ? up(rows * q_heads * width * 4) : 0;
    s.total = s.part + s.ml + s.stat + s.scores;
    return s;
}

template <typename T, int D, int GP>
int launch_attention(AttnArgs a, float *weights, size_t w_row, size_t w_head, cudaStream_t st) {
    const int smem = attn_smem<T, D, GP>(), blocks = attn_blocks();
    FOCR_CUDA_TRY(set_max_dynamic_smem((const void *)paged_attention_kernel<T, D, GP>, smem));
    a.head_chunks = (a.group + GP - 1) / GP;
    FOCR_CUDA_TRY(launch_pdl(paged_attention_kernel<T, D, GP>, blocks, WARPS * 32, smem, st, a));
    const dim3 grid(a.c.kv_heads * a.head_chunks, a.rows);
    FOCR_CUDA_TRY(launch_pdl(paged_join_kernel<Tile<T, D>::BLOCK, GP>, grid, WARPS * 32, 0, st, a, blocks));
    if (weights) {
        const dim3 wgrid((a.width + 255) / 256, a.c.kv_heads, a.rows);
        FOCR_CUDA_TRY(launch_pdl(paged_weights_kernel, wgrid, 256, 0, st, a, weights,
                                 (long long)w_row, (long long)w_head));
    }
    return FOCR_OK;
}

template <typename T, int D>
int by_group(const AttnArgs &a, float *w, size_t wr, size_t wh, cudaStream_t st) {
    switch (heads_together(a.group)) {
        case 1: return launch_attention<T, D, 1>(a, w, wr, wh, st);
        case 2: return launch_attention<T, D, 2>(a, w, wr, wh, st);
        case 4: return launch_attention<T, D, 4>(a, w, wr, wh, st);
        default: return launch_attention<T, D, 8>(a, w, wr, wh, st);
    }
}
template <typename T>
int by_dim(const AttnArgs &a, float *w, size_t wr, size_t wh, cudaStream_t st) {
    return a.dim <= 64 ? by_group<T, 64>(a, w, wr, wh, st)
         : a.dim <= 128 ? by_group<T, 128>(a, w, wr, wh, st)
                        : by_group<T, 256>(a, w, wr, wh, st);
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" {

int focr_paged_attention_workspace(size_t rows, size_t q_heads, size_t head_dim,
                                   size_t weights_width, size_t *bytes) {
    return guarded("paged_attention_workspace", [&]() -> int {
        if (!bytes) return fail(FOCR_E_ARG, "paged_attention_workspace: null pointer");
        size_t n;
        if (!checked_mul(rows, q_heads, &n) || !checked_mul(n, weights_width, &n) || n > SIZE_MAX / 16)
            return fail(FOCR_E_SHAPE, "paged_attention_workspace: size overflow");
        *bytes = attn_sizes(rows, q_heads, head_dim, weights_width).total;
        return FOCR_OK;
    });
}

int focr_paged_attention(const focr_paged_cache *cache, const void *q, int q_dtype, size_t rows,
                         size_t q_heads, size_t q_stride, const int32_t *lens,
                         const int32_t *ref_lens, size_t window, float scale, void *out,
                         size_t out_stride, float *weights, size_t weights_width,
                         size_t weights_row_stride, size_t weights_head_stride, void *workspace,
                         size_t workspace_bytes, void *stream) {
    return guarded("paged_attention", [&]() -> int {
        AttnArgs a{};
        int rc = paged_view("paged_attention", cache, rows, &a.c);
        if (rc) return rc;
        if (q_dtype != FOCR_F32 && q_dtype != FOCR_F16 && q_dtype != FOCR_BF16)
            return fail(FOCR_E_ARG, "paged_attention: unknown query type " + std::to_string(q_dtype));
        if (q_heads == 0 || q_heads % cache->kv_heads || q_heads > INT32_MAX)
            return fail(FOCR_E_SHAPE, "paged_attention: " + std::to_string(q_heads) +
                                          " query heads over " + std::to_string(cache->kv_heads) +
                                          " kv heads");
        if (!(scale > 0.0f) || !std::isfinite(scale))
            return fail(FOCR_E_ARG, "paged_attention: scale must be positive and finite");
        if (rows == 0) return FOCR_OK;
        if (!q || !lens || !out || !workspace) return fail(FOCR_E_ARG, "paged_attention: null pointer");
        if (rows > INT32_MAX) return fail(FOCR_E_UNSUPPORTED, "paged_attention: dimension exceeds int32 range");
        const size_t wide = q_heads * cache->head_dim;
        if (rows > 1 && (q_stride < wide || out_stride < wide))
            return fail(FOCR_E_SHAPE, "paged_attention: a row stride is shorter than q_heads * head_dim");
        if (q_stride > (size_t)INT64_MAX / 8 / rows || out_stride > (size_t)INT64_MAX / 8 / rows)
            return fail(FOCR_E_SHAPE, "paged_attention: stride overflow");
        const size_t cap = (size_t)cache->max_pages * cache->page_size;
        if (weights) {
            if (weights_width == 0 || weights_width > INT32_MAX)
                return fail(FOCR_E_SHAPE, "paged_attention: weights_width out of range");
            if ((cache->kv_heads > 1 && weights_head_stride < weights_width) ||
                (rows > 1 && weights_row_stride < weights_width))
                return fail(FOCR_E_SHAPE, "paged_attention: a weights stride is shorter than weights_width");
        }
        if (cache->kv_heads > 65535)
            return fail(FOCR_E_UNSUPPORTED, "paged_attention: over 65535 kv heads");
        const size_t width = weights ? (weights_width < cap ? weights_width : cap) : 0;
        const Sizes sz = attn_sizes(rows < MAX_ROWS ? rows : MAX_ROWS, q_heads, cache->head_dim, width);
        if (workspace_bytes < sz.total || (uintptr_t)workspace % 16)
            return fail(FOCR_E_ARG, "paged_attention: the workspace needs " + std::to_string(sz.total) +
                                        " bytes, 16-byte aligned");
        char *ws = (char *)workspace;
        a.part = (float *)ws;
        a.ml = (float2 *)(ws + sz.part);
        if (weights) {
            a.stat = (float2 *)(ws + sz.part + sz.ml);
            a.scores = (float *)(ws + sz.part + sz.ml + sz.stat);
        }
        a.q_stride = (long long)q_stride;
        a.out_stride = (long long)out_stride;
        a.q_heads = (int)q_heads;
        a.group = (int)(q_heads / cache->kv_heads);
        a.dim = (int)cache->head_dim;
        a.q_type = q_dtype;
        a.window = window > INT32_MAX ? 0 : (int)window;
        a.width = (int)width;
        a.cap = weights ? (int)width : (int)cap;
        a.c2 = (float)(scale * 1.4426950408889634);
        const size_t q_size = dtype_bytes(q_dtype);
        for (size_t r0 = 0; r0 < rows; r0 += MAX_ROWS) {
            AttnArgs b = a;
            b.rows = (int)(rows - r0 < MAX_ROWS ? rows - r0 : MAX_ROWS);
            b.c.table += r0 * cache->table_stride;
            b.q = (const char *)q + r0 * q_stride * q_size;
            b.out = (char *)out + r0 * out_stride * q_size;
            b.lens = lens + r0;
            b.refs = ref_lens ? ref_lens + r0 : nullptr;
            float *w = weights ? weights + r0 * weights_row_stride : nullptr;
            cudaStream_t st = (cudaStream_t)stream;
            rc = cache->dtype == FOCR_F32 ? by_dim<float>(b, w, weights_row_stride, weights_head_stride, st)
               : cache->dtype == FOCR_F16 ? by_dim<__half>(b, w, weights_row_stride, weights_head_stride, st)
                                          : by_dim<__nv_bfloat16>(b, w, weights_row_stride, weights_head_stride, st);
            if (rc) return rc;
        }
        return FOCR_OK;
    });
}

}  // extern "C"
