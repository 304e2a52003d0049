// Attention of one new token per row over a paged cache: the join of the pieces,
// the accumulated weights, and the entry point.
#include "paged_attention.cuh"

namespace focr {
namespace {

constexpr int JT = 256;

// Joins the pieces of the (row, kv head, chunk of query heads)s that block
// boundaries cut: a block per boundary, of which the one at a cut's first boundary
// does the work, for `heads` query heads of the chunk.  Where a (row, head) can have few
// pieces a warp joins a head.  A long row of a small batch has pieces of nearly every
// block: there a block has one head, the pieces' factors are found side by side first,
// and the threads split the pieces as well as the columns.  Latency bounds it: some 3 us
// behind the attention kernel, whose end it overlaps up to its lengths' prefix.
__global__ void __launch_bounds__(JT) paged_join_kernel(const AttnArgs a, int blocks, int heads) {
    extern __shared__ float factor[];   // [pieces]
    __shared__ int pre[ATTN_ROWS + 1];
    __shared__ float4 red[JT];
    __shared__ float warp_m[JT / 32], warp_l[JT / 32];
    // the kernel before has waited for all that came before it: lengths may be
    // read while it still runs
    tile_prefix<JT>(a, pre);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, HC = a.c.kv_heads * a.head_chunks;
    const unsigned long long total = (unsigned long long)pre[a.rows] * HC, n = run_count(total, blocks);
    const unsigned long long b = blockIdx.x + 1;
    pdl_wait();
    pdl_trigger();
    if (b >= n) return;
    const unsigned long long u = quotient(b * total, n), before = quotient((b - 1) * total, n);
    const int r = row_of_unit(pre, a.rows, HC, u), tiles = pre[r + 1] - pre[r];
    const int hc = (int)quotient(u - (unsigned long long)pre[r] * HC, tiles);
    const unsigned long long u0 = (unsigned long long)pre[r] * HC + (unsigned long long)hc * tiles;
    if (u == u0 || before > u0) return;   // nothing is cut, or it was cut before
    const int kvh = hc / a.head_chunks, g0 = (hc - kvh * a.head_chunks) * a.gp;
    // the last block whose run begins before the cut ends
    const int b0 = (int)b - 1, b1 = (int)quotient((u0 + tiles) * n - 1, total);
    const int pieces = b1 - b0 + 1, slot0 = 2 * b0 + (before == u0 ? 0 : 1);
    auto slot = [&](int p) { return p ? 2 * (b0 + p) : slot0; };
    const int columns = a.dim / 4;   // at most 64
    const int g_end = min(min(a.gp, a.group - g0), (int)(blockIdx.y + 1) * heads);
    if (heads > 1 && pieces <= 32) {   // a warp a head
        for (int g = blockIdx.y * heads + warp; g < g_end; g += JT / 32) {
            const float2 ml = lane < pieces ? a.ml[slot(lane) * a.gp + g] : make_float2(-INFINITY, 0.0f);
            const float M = warp_max_f32(ml.x), f = lane < pieces ? rescale(ml.x, M, a.c2) : 0.0f;
            float L = ml.y * f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
            if (a.stat && lane == 0) a.stat[(int64_t)r * a.q_heads + kvh * a.group + g0 + g] = make_float2(M, 1.0f / L);
            float4 o[2] = {};
#pragma unroll 4
            for (int p = 0; p < pieces; p++) {
                const float fp = __shfl_sync(0xffffffffu, f, p);
                const float4 *x = reinterpret_cast<const float4 *>(a.part + ((int64_t)slot(p) * a.gp + g) * a.dim);
#pragma unroll
                for (int y = 0; y < 2; y++)
                    if (lane + y * 32 < columns) o[y] = fma4(x[lane + y * 32], fp, o[y]);
            }
#pragma unroll
            for (int y = 0; y < 2; y++)
                if (lane + y * 32 < columns)
                    store4_as(a.out, a.q_type, r * a.out_stride + (long long)(kvh * a.group + g0 + g) * a.dim + 4 * (lane + y * 32),
                              over4(o[y], L, true));
        }
        return;
    }
    for (int g = blockIdx.y * heads; g < g_end; g++) {
        const int qh = kvh * a.group + g0 + g;
        float M = -INFINITY, L = 0.0f;
        for (int p = t; p < pieces; p += JT) M = fmaxf(M, a.ml[slot(p) * a.gp + g].x);
        M = warp_max_f32(M);
        if (lane == 0) warp_m[warp] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < JT / 32; w++) M = fmaxf(M, warp_m[w]);
        for (int p = t; p < pieces; p += JT) {
            const float2 ml = a.ml[slot(p) * a.gp + g];
            const float f = rescale(ml.x, M, a.c2);
            factor[p] = f;
            L = __fmaf_rn(ml.y, f, L);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane == 0) warp_l[warp] = L;
        __syncthreads();
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < JT / 32; w++) L += warp_l[w];
        if (a.stat && t == 0) a.stat[(int64_t)r * a.q_heads + qh] = make_float2(M, 1.0f / L);
        int ct = 8;
        while (ct < columns) ct <<= 1;
        const int splits = JT / ct, part = t / ct, c = t % ct;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c < columns)
#pragma unroll 4
            for (int p = part; p < pieces; p += splits)
                o = fma4(reinterpret_cast<const float4 *>(a.part + ((int64_t)slot(p) * a.gp + g) * a.dim)[c], factor[p], o);
        red[t] = o;
        __syncthreads();
        if (!part && c < columns) {
            for (int s = 1; s < splits; s++) o = fma4(red[t + s * ct], 1.0f, o);
            store4_as(a.out, a.q_type, r * a.out_stride + (long long)qh * a.dim + 4 * c, over4(o, L, true));
        }
    }
}

// weights[r][kv head][j] += sum over the kv head's query heads of p_j, from the
// kept scores.  Where one of them has no probabilities the weights stay as they were.  Bound by
// the scores' bytes, most of them still in L2: 32 rows of 8300 positions on average,
// 8 kv heads with 4 query heads each: 13.5 us for 51 MB (22.8 with one position a
// thread).
__global__ void __launch_bounds__(256) paged_weights_kernel(const AttnArgs a, float *weights,
                                                            long long w_row, long long w_head) {
    constexpr int U = 4;   // positions of a thread, loaded together
    __shared__ float2 st[256];
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y, t = threadIdx.x;
    const RowView rv = row_view(a, r);
    const int i0 = blockIdx.x * (256 * U) + t;
    if (i0 - t >= rv.vis) return;
    float *w = weights + r * w_row + kvh * w_head;
    float sum[U], old[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * 256;
        old[u] = i < rv.vis ? w[i < rv.ref ? i : i + rv.gap] : 0.0f;
        sum[u] = 0.0f;
    }
    for (int g0 = 0; g0 < a.group; g0 += 256) {
        const int heads = min(256, a.group - g0);
        __syncthreads();
        if (t < heads) {   // (M, 1 / L)
            const float2 x = a.stat[(int64_t)r * a.q_heads + kvh * a.group + g0 + t];
            st[t] = make_float2(base_of(x.x), x.y);
        }
        __syncthreads();
        const float *s = a.scores + ((int64_t)r * a.q_heads + kvh * a.group + g0) * a.score_stride;
#pragma unroll 2
        for (int g = 0; g < heads; g++) {
            float x[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                x[u] = i0 + u * 256 < rv.vis ? s[(int64_t)g * a.score_stride + i0 + u * 256] : -INFINITY;
#pragma unroll
            for (int u = 0; u < U; u++) sum[u] = __fmaf_rn(prob(x[u], a.c2, st[g].x), st[g].y, sum[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = i0 + u * 256;
        if (i < rv.vis && isfinite(sum[u])) w[i < rv.ref ? i : i + rv.gap] = old[u] + sum[u];
    }
}

struct Sizes {
    size_t scores, stat, part, ml, total;
};
Sizes attn_sizes(size_t rows, size_t q_heads, size_t dim, size_t width) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    Sizes s;
    const size_t slots = (size_t)attn_blocks() * 2 * ATTN_HEADS;
    s.part = up(slots * dim * 4);
    s.ml = up(slots * 8);
    s.stat = width ? up(rows * q_heads * 8) : 0;
    s.scores = width ? up(rows * q_heads * ((width + 1) & ~(size_t)1) * 4) : 0;
    s.total = s.part + s.ml + s.stat + s.scores;
    return s;
}

int launch_attention(AttnArgs a, int dtype, float *weights, size_t w_row, size_t w_head, cudaStream_t st) {
    const int rc = dtype == FOCR_F32   ? launch_attention_f32(a, st)
                   : dtype == FOCR_F16 ? launch_attention_f16(a, st)
                                       : launch_attention_bf16(a, st);
    if (rc) return rc;
    const int blocks = attn_blocks();
    if (a.cluster == RUNS && blocks > 1) {
        const int most = a.gp < a.group ? a.gp : a.group;
        const int heads = most == 1 || (size_t)a.rows * a.c.kv_heads * a.head_chunks * 8 < (size_t)blocks ? 1 : 8;
        FOCR_CUDA_TRY(launch_pdl(paged_join_kernel, dim3(blocks - 1, (most + heads - 1) / heads), JT, blocks * 4, st, a, blocks, heads));
    }
    if (weights)
        FOCR_CUDA_TRY(launch_pdl(paged_weights_kernel, dim3((a.width + 1023) / 1024, a.c.kv_heads, a.rows), 256, 0, st,
                                 a, weights, (long long)w_row, (long long)w_head));
    return FOCR_OK;
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
        *bytes = attn_sizes(rows < ATTN_ROWS ? rows : ATTN_ROWS, q_heads, head_dim, weights_width).total;
        return FOCR_OK;
    });
}

int focr_paged_attention(const focr_paged_cache *cache, const focr_paged_attention_args *args, void *stream) {
    return guarded("paged_attention", [&]() -> int {
        if (!args) return fail(FOCR_E_ARG, "paged_attention: null arguments");
        const void *q = args->q;
        const int32_t *lens = args->lens;
        const int32_t *ref_lens = args->ref_lens;
        void *out = args->out;
        float *weights = args->weights;
        void *workspace = args->workspace;
        const size_t rows = args->rows;
        const size_t q_heads = args->q_heads;
        const size_t q_stride = args->q_stride;
        const size_t out_stride = args->out_stride;
        const size_t window = args->window;
        const size_t weights_width = args->weights_width;
        const size_t weights_row_stride = args->weights_row_stride;
        const size_t weights_head_stride = args->weights_head_stride;
        const size_t workspace_bytes = args->workspace_bytes;
        const int q_dtype = args->q_dtype;
        const float scale = args->scale;
        AttnArgs a{};
        int rc = paged_view("paged_attention", cache, rows, &a.c);
        if (rc) return rc;
        if (q_dtype != FOCR_F32 && q_dtype != FOCR_F16 && q_dtype != FOCR_BF16)
            return fail(FOCR_E_ARG, "paged_attention: unknown query type " + std::to_string(q_dtype));
        if (q_heads == 0 || q_heads % cache->kv_heads || q_heads > (1u << 20))
            return fail(FOCR_E_SHAPE, "paged_attention: " + std::to_string(q_heads) +
                                          " query heads over " + std::to_string(cache->kv_heads) +
                                          " kv heads");
        a.c2 = (float)(scale * 1.4426950408889634);
        if (!(a.c2 > 0.0f) || !std::isfinite(a.c2))
            return fail(FOCR_E_ARG, "paged_attention: scale must be positive and finite");
        if (rows == 0) return FOCR_OK;
        if (!q || !lens || !out || !workspace) return fail(FOCR_E_ARG, "paged_attention: null pointer");
        if (out == q) return fail(FOCR_E_ARG, "paged_attention: out must not be q");
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
        const Sizes sz = attn_sizes(rows < ATTN_ROWS ? rows : ATTN_ROWS, q_heads, cache->head_dim, width);
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
        a.score_stride = (int)((width + 1) & ~(size_t)1);
        a.cap = weights ? (int)width : (int)cap;
        const size_t q_size = dtype_bytes(q_dtype);
        const size_t most = (size_t)attn_rows((size_t)a.cap);
        for (size_t r0 = 0; r0 < rows; r0 += most) {
            AttnArgs b = a;
            b.rows = (int)(rows - r0 < most ? rows - r0 : most);
            b.c.table += r0 * cache->table_stride;
            b.q = (const char *)q + r0 * q_stride * q_size;
            b.out = (char *)out + r0 * out_stride * q_size;
            b.lens = lens + r0;
            b.refs = ref_lens ? ref_lens + r0 : nullptr;
            float *w = weights ? weights + r0 * weights_row_stride : nullptr;
            cudaStream_t st = (cudaStream_t)stream;
            rc = launch_attention(b, cache->dtype, w, weights_row_stride, weights_head_stride, st);
            if (rc) return rc;
        }
        return FOCR_OK;
    });
}

}  // extern "C"
