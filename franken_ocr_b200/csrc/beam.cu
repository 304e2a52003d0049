// Beam search over the decoder's logits: the choice of the next beams
// (focr_beam_select) and the reordering of their pages (focr_beam_reorder).
//
// A candidate (beam i, token t) scores
//   cum_i + ((x_t - m_i) - log sum_u exp(x_u - m_i)),   m_i = max_u x_u,
// and candidates are ranked by score, then lower beam, then larger logit, then
// lower token.  The sum and the scores are held in 64 bits: candidates of
// different beams often lie closer than f32 resolves, and a choice, unlike a
// value, cannot be a little off.
//
// Within one beam the ranking is the logits' own, so no sum is needed to
// shorten the list: select_part_kernel reads each vocabulary strip once and
// keeps its sum and its n largest logits; select_join_kernel, a block per
// entry, has beams * strips * n candidates left to rank.
#include "paged.cuh"

namespace focr {
namespace {

constexpr int ST = 256;              // threads of both kernels
constexpr int PER = 32;              // logits a thread of a strip
constexpr int STRIP = ST * PER;
constexpr int MAX_N = 64;

struct SelectArgs {
    const void *x;
    const float *cum;
    const uint8_t *done;
    float *score_out;
    int32_t *parent_out, *token_out;
    long long row_stride;            // elements between the logits of two beams
    int beams, vocab, n, strips, end_token;
    // workspace, per (row, strip): n (logit, token) pairs, (max, sum)
    float *cx;
    int32_t *ct;
    float *pm;
    double *ps;
};

// Order-preserving bits of a logit; NaN and -inf are no candidates (0), +inf
// counts as the largest finite value.
__device__ __forceinline__ uint32_t logit_key(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(fminf(x, 3.402823466e38f) + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ uint64_t warp_max_u64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}

// The strip's largest key below `below`, over the block.
__device__ uint64_t block_max_u64(uint64_t v, uint64_t *sh) {
    v = warp_max_u64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    uint64_t m = sh[0];
#pragma unroll
    for (int w = 1; w < ST / 32; w++) m = sh[w] > m ? sh[w] : m;
    return m;
}

template <typename T>
__global__ void __launch_bounds__(ST) select_part_kernel(const SelectArgs a) {
    __shared__ uint64_t sh[ST / 32];
    __shared__ double shd[ST / 32];
    pdl_wait();
    pdl_trigger();
    const int strip = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.row_stride;
    const int first = strip * STRIP;
    uint32_t key[PER];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int c = first + i * ST + t;
        key[i] = c < a.vocab ? logit_key(to_f32<T>(x[c])) : 0;
        top = max(top, key[i]);
    }
    const uint32_t m = (uint32_t)block_max_u64(top, sh);
    const double mx = key_logit(m);
    double sum = 0.0;
    if (m)
#pragma unroll 1
        for (int i = 0; i < PER; i++)
            if (key[i]) sum += exp((double)key_logit(key[i]) - mx);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((t & 31) == 0) shd[t >> 5] = sum;
    __syncthreads();
    const long long at = (long long)row * a.strips + strip;
    if (t == 0) {
        for (int w = 1; w < ST / 32; w++) sum += shd[w];
        a.pm[at] = m ? key_logit(m) : -INFINITY;
        a.ps[at] = sum;
    }
    // the n largest, one after the other: (key, ~token) as one number
    uint64_t below = ~0ull;
    for (int k = 0; k < a.n; k++) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint64_t v = (uint64_t)key[i] << 32 | (uint32_t)~(first + i * ST + t);
            if (key[i] && v < below && v > best) best = v;
        }
        best = block_max_u64(best, sh);
        if (t == 0) {
            a.cx[at * a.n + k] = best ? key_logit((uint32_t)(best >> 32)) : -INFINITY;
            a.ct[at * a.n + k] = best ? (int32_t)~(uint32_t)best : -1;
        }
        below = best;
        if (!best) below = 0;
    }
}

struct Cand {
    double score;
    float x;
    int beam, token;
};
__device__ __forceinline__ bool before(const Cand &p, const Cand &q) {  // p ranks above q
    if (p.score != q.score) return p.score > q.score;
    if (p.beam != q.beam) return p.beam < q.beam;
    if (p.x != q.x) return p.x > q.x;
    return p.token < q.token;
}

__global__ void __launch_bounds__(ST) select_join_kernel(const SelectArgs a) {
    __shared__ double lse_m[MAX_N], lse_s[MAX_N];
    __shared__ Cand best[ST / 32];
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.x, t = threadIdx.x;
    for (int i = t; i < a.beams; i += ST) {
        const long long row = (long long)b * a.beams + i;
        float m = -INFINITY;
        for (int s = 0; s < a.strips; s++) m = fmaxf(m, a.pm[row * a.strips + s]);
        double sum = 0.0;
        for (int s = 0; s < a.strips; s++) {
            const float p = a.pm[row * a.strips + s];
            if (p > -INFINITY) sum += a.ps[row * a.strips + s] * exp((double)p - (double)m);
        }
        lse_m[i] = m;
        lse_s[i] = log(sum);
    }
    __syncthreads();
    const int per = a.strips * a.n, total = a.beams * per;
    Cand last{INFINITY, INFINITY, -1, -1};
    for (int k = 0; k < a.n; k++) {
        Cand mine{-INFINITY, -INFINITY, INT_MAX, INT_MAX};
        for (int j = t; j < total; j += ST) {
            const int beam = j / per, rest = j - beam * per;
            const long long row = (long long)b * a.beams + beam;
            const float cum = a.cum[row];
            if (!isfinite(cum)) continue;
            Cand c;
            c.beam = beam;
            if (a.done && a.done[row]) {
                if (rest) continue;
                c.score = cum;
                c.x = 0.0f;
                c.token = a.end_token;
            } else {
                c.x = a.cx[row * per + rest];
                c.token = a.ct[row * per + rest];
                if (c.token < 0) continue;
                c.score = (double)cum + (((double)c.x - lse_m[beam]) - lse_s[beam]);
            }
            if ((k == 0 || before(last, c)) && before(c, mine)) mine = c;
        }
        for (int o = 16; o > 0; o >>= 1) {
            Cand c;
            c.score = __shfl_xor_sync(0xffffffffu, mine.score, o);
            c.x = __shfl_xor_sync(0xffffffffu, mine.x, o);
            c.beam = __shfl_xor_sync(0xffffffffu, mine.beam, o);
            c.token = __shfl_xor_sync(0xffffffffu, mine.token, o);
            if (before(c, mine)) mine = c;
        }
        __syncthreads();
        if ((t & 31) == 0) best[t >> 5] = mine;
        __syncthreads();
        last = best[0];
        for (int w = 1; w < ST / 32; w++)
            if (before(best[w], last)) last = best[w];
        if (t == 0) {
            const bool have = last.beam != INT_MAX;
            const long long o = (long long)b * a.n + k;
            a.score_out[o] = have ? (float)last.score : -INFINITY;
            a.parent_out[o] = have ? last.beam : -1;
            a.token_out[o] = have ? last.token : -1;
        }
    }
}

struct SelectSizes {
    size_t cx, ct, pm, ps, total;
};
SelectSizes select_sizes(size_t rows, size_t vocab, size_t n) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t parts = rows * ((vocab + STRIP - 1) / STRIP);
    SelectSizes s;
    s.cx = up(parts * n * 4);
    s.ct = up(parts * n * 4);
    s.pm = up(parts * 4);
    s.ps = up(parts * 8);
    s.total = s.cx + s.ct + s.pm + s.ps;
    return s;
}

// ---- reordering -----------------------------------------------------------

struct ReorderArgs {
    PagedView c;
    const int32_t *lens, *parent, *fresh;
    int32_t *table_out, *lens_out;
    const float *w;
    float *w_out;
    int64_t layer_stride;   // bytes between two layers' pages
    long long w_layer, w_row, w_head, wo_layer;
    int rows, beams, layers, width;
};

__device__ __forceinline__ int reorder_source(const ReorderArgs &a, int i) {
    const int p = a.parent[i];
    return p < 0 || p >= a.beams ? -1 : i / a.beams * a.beams + p;
}
__device__ __forceinline__ int reorder_len(const ReorderArgs &a, int src) {
    const int n = src < 0 ? 0 : a.lens[src];
    return n < 0 || n > a.c.max_pages * a.c.page_size ? 0 : n;
}

// A block per (row, layer and kv head): the partly filled page's slots, and the
// weights; the blocks of the first layer and head also write the row's table.
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderArgs a) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.y, lh = blockIdx.x, t = threadIdx.x;
    const int layer = lh / a.c.kv_heads, h = lh - layer * a.c.kv_heads;
    const int src = reorder_source(a, i), n = reorder_len(a, src);
    const int full = n / a.c.page_size, rest = n - full * a.c.page_size;
    const int32_t *pages = a.c.table + (int64_t)(src < 0 ? 0 : src) * a.c.table_stride;
    const int here = a.fresh[i];
    if (lh == 0) {
        for (int j = t; j < a.c.max_pages; j += 256)
            a.table_out[(int64_t)i * a.c.max_pages + j] = j < full ? pages[j] : j == full ? here : -1;
        if (t == 0) a.lens_out[i] = n;
    }
    if (rest > 0) {
        const int from = pages[full];
        if ((uint32_t)from < (uint32_t)a.c.n_pages && (uint32_t)here < (uint32_t)a.c.n_pages) {
            const int64_t at = layer * a.layer_stride + h * a.c.head_stride;
            const int64_t s = at + from * a.c.page_stride, d = at + here * a.c.page_stride;
            for (int x = t; x < rest * (a.c.row_bytes / 16); x += 256) {
                ((uint4 *)(a.c.k + d))[x] = ((const uint4 *)(a.c.k + s))[x];
                ((uint4 *)(a.c.v + d))[x] = ((const uint4 *)(a.c.v + s))[x];
            }
        }
    }
    if (a.w) {
        const float *w = a.w + layer * a.w_layer + (src < 0 ? 0 : src) * a.w_row + h * a.w_head;
        float *o = a.w_out + layer * a.wo_layer + ((int64_t)i * a.c.kv_heads + h) * a.width;
        for (int x = t; x < a.width; x += 256) o[x] = x < n ? w[x] : 0.0f;
    }
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" {

int focr_beam_select_workspace(size_t batch, size_t beams, size_t vocab, size_t n, size_t *bytes) {
    return guarded("beam_select_workspace", [&]() -> int {
        if (!bytes) return fail(FOCR_E_ARG, "beam_select_workspace: null pointer");
        size_t rows, x;
        if (!checked_mul(batch, beams, &rows) || !checked_mul(rows, vocab / STRIP + 1, &x) || n > MAX_N ||
            x > SIZE_MAX / 1024)
            return fail(FOCR_E_SHAPE, "beam_select_workspace: size out of range");
        *bytes = select_sizes(rows, vocab, n).total;
        return FOCR_OK;
    });
}

int focr_beam_select(const void *logits, int dtype, size_t batch, size_t beams, size_t vocab,
                     size_t row_stride, const float *scores, const uint8_t *done, int32_t end_token,
                     size_t n, float *scores_out, int32_t *parent_out, int32_t *token_out,
                     void *workspace, size_t workspace_bytes, void *stream) {
    return guarded("beam_select", [&]() -> int {
        if (dtype != FOCR_F32 && dtype != FOCR_F16 && dtype != FOCR_BF16)
            return fail(FOCR_E_ARG, "beam_select: unknown logits type " + std::to_string(dtype));
        if (beams == 0 || vocab == 0 || n == 0)
            return fail(FOCR_E_SHAPE, "beam_select: beams, vocab and n must not be 0");
        if (beams > MAX_N || n > MAX_N)
            return fail(FOCR_E_UNSUPPORTED, "beam_select: beams and n are at most " + std::to_string(MAX_N));
        if (vocab > (size_t)INT32_MAX - STRIP || batch > (size_t)65535 / beams)
            return fail(FOCR_E_UNSUPPORTED, "beam_select: over 65535 rows, or vocab exceeds int32 range");
        if (batch == 0) return FOCR_OK;
        if (batch * beams > 1 && row_stride < vocab)
            return fail(FOCR_E_SHAPE, "beam_select: row_stride " + std::to_string(row_stride) +
                                          " < vocab " + std::to_string(vocab));
        if (row_stride > (size_t)INT64_MAX / 8 / (batch * beams))
            return fail(FOCR_E_SHAPE, "beam_select: stride overflow");
        if (!logits || !scores || !scores_out || !parent_out || !token_out || !workspace)
            return fail(FOCR_E_ARG, "beam_select: null pointer");
        const SelectSizes sz = select_sizes(batch * beams, vocab, n);
        if (workspace_bytes < sz.total || (uintptr_t)workspace % 16)
            return fail(FOCR_E_ARG, "beam_select: the workspace needs " + std::to_string(sz.total) +
                                        " bytes, 16-byte aligned");
        SelectArgs a{};
        a.x = logits;
        a.cum = scores;
        a.done = done;
        a.score_out = scores_out;
        a.parent_out = parent_out;
        a.token_out = token_out;
        a.row_stride = (long long)row_stride;
        a.beams = (int)beams;
        a.vocab = (int)vocab;
        a.n = (int)n;
        a.strips = (int)((vocab + STRIP - 1) / STRIP);
        a.end_token = end_token;
        char *ws = (char *)workspace;
        a.ps = (double *)ws;
        a.cx = (float *)(ws + sz.ps);
        a.ct = (int32_t *)(ws + sz.ps + sz.cx);
        a.pm = (float *)(ws + sz.ps + sz.cx + sz.ct);
        cudaStream_t st = (cudaStream_t)stream;
        const dim3 grid(a.strips, (unsigned)(batch * beams));
        auto *part = dtype == FOCR_F32 ? select_part_kernel<float>
                   : dtype == FOCR_F16 ? select_part_kernel<__half>
                                       : select_part_kernel<__nv_bfloat16>;
        FOCR_CUDA_TRY(launch_pdl(part, grid, ST, 0, st, a));
        FOCR_CUDA_TRY(launch_pdl(select_join_kernel, (unsigned)batch, ST, 0, st, a));
        return FOCR_OK;
    });
}

int focr_beam_reorder(const focr_paged_cache *cache, size_t layers, size_t layer_stride,
                      size_t batch, size_t beams, const int32_t *lens, const int32_t *parent,
                      const int32_t *fresh, int32_t *table_out, int32_t *lens_out,
                      const float *weights, size_t width, size_t weights_layer_stride,
                      size_t weights_row_stride, size_t weights_head_stride, float *weights_out,
                      void *stream) {
    return guarded("beam_reorder", [&]() -> int {
        ReorderArgs a{};
        size_t rows;
        if (!checked_mul(batch, beams, &rows)) return fail(FOCR_E_SHAPE, "beam_reorder: batch*beams overflow");
        int rc = paged_view("beam_reorder", cache, rows, &a.c);
        if (rc) return rc;
        if (beams == 0 || layers == 0) return fail(FOCR_E_SHAPE, "beam_reorder: beams and layers must not be 0");
        if (rows == 0) return FOCR_OK;
        if (!lens || !parent || !fresh || !table_out || !lens_out)
            return fail(FOCR_E_ARG, "beam_reorder: null pointer");
        size_t lh;
        if (rows > 65535 || !checked_mul(layers, cache->kv_heads, &lh) || lh > INT32_MAX || width > INT32_MAX)
            return fail(FOCR_E_UNSUPPORTED, "beam_reorder: dimension out of range");
        const size_t size = dtype_bytes(cache->dtype);
        if (layers > 1 && (layer_stride < (size_t)cache->page_size * cache->head_dim ||
                           layer_stride > (size_t)INT64_MAX / size / layers || layer_stride * size % 16))
            return fail(FOCR_E_SHAPE, "beam_reorder: bad layer stride");
        if (table_out == cache->table || lens_out == lens)
            return fail(FOCR_E_ARG, "beam_reorder: the outputs must not be the inputs");
        if (weights) {
            if (!weights_out || weights_out == weights)
                return fail(FOCR_E_ARG, "beam_reorder: weights_out must be there and not be weights");
            if (width == 0 || (cache->kv_heads > 1 && weights_head_stride < width) ||
                (rows > 1 && weights_row_stride < width) || (layers > 1 && weights_layer_stride < width))
                return fail(FOCR_E_SHAPE, "beam_reorder: a weights stride is shorter than the width");
        }
        a.lens = lens;
        a.parent = parent;
        a.fresh = fresh;
        a.table_out = table_out;
        a.lens_out = lens_out;
        a.w = weights;
        a.w_out = weights_out;
        a.layer_stride = layers > 1 ? (int64_t)(layer_stride * size) : 0;
        a.w_layer = (long long)weights_layer_stride;
        a.w_row = (long long)weights_row_stride;
        a.w_head = (long long)weights_head_stride;
        a.wo_layer = (long long)rows * cache->kv_heads * (long long)width;
        a.rows = (int)rows;
        a.beams = (int)beams;
        a.layers = (int)layers;
        a.width = (int)width;
        FOCR_CUDA_TRY(launch_pdl(beam_reorder_kernel, dim3((unsigned)lh, (unsigned)rows), 256, 0,
                                 (cudaStream_t)stream, a));
        return FOCR_OK;
    });
}

}  // extern "C"
