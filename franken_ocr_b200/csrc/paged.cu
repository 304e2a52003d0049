// Paged K/V cache: the checks every call on a cache makes, and the write of
// new keys and values into pages.
#include "paged.cuh"

namespace focr {

int paged_view(const char *ctx, const focr_paged_cache *c, size_t rows, PagedView *out) {
    const std::string at = std::string(ctx) + ": ";
    if (!c) return fail(FOCR_E_ARG, at + "null cache");
    if (c->dtype != FOCR_F32 && c->dtype != FOCR_F16 && c->dtype != FOCR_BF16)
        return fail(FOCR_E_ARG, at + "unknown cache type " + std::to_string(c->dtype));
    if (!c->n_pages || !c->kv_heads || !c->page_size || !c->head_dim || !c->max_pages)
        return fail(FOCR_E_SHAPE, at + "the cache has an empty dimension");
    if (c->n_pages > INT32_MAX || c->kv_heads > INT32_MAX)
        return fail(FOCR_E_UNSUPPORTED, at + "dimension exceeds int32 range");
    const size_t size = dtype_bytes(c->dtype);
    if (c->head_dim > 256 || c->head_dim * size % 16)
        return fail(FOCR_E_UNSUPPORTED, at + "head_dim " + std::to_string(c->head_dim) +
                                            " is over 256 or not a multiple of 16 bytes");
    if ((uint64_t)c->max_pages * c->page_size > (uint64_t)INT32_MAX - 65535)   // room for whole tiles
        return fail(FOCR_E_UNSUPPORTED, at + "max_pages * page_size exceeds int32 range");
    const size_t rows_bytes = (size_t)c->page_size * c->head_dim;
    if (c->page_stride > (size_t)INT64_MAX / size / c->n_pages ||
        c->head_stride > (size_t)INT64_MAX / size / c->kv_heads)
        return fail(FOCR_E_SHAPE, at + "stride overflow");
    if (c->page_stride * size % 16 || c->head_stride * size % 16)
        return fail(FOCR_E_UNSUPPORTED, at + "page and head strides are multiples of 16 bytes");
    if ((c->kv_heads > 1 && c->head_stride < rows_bytes) ||
        (c->n_pages > 1 && c->page_stride < rows_bytes))
        return fail(FOCR_E_SHAPE, at + "a stride is shorter than page_size * head_dim");
    if (rows > 1 && c->table_stride < c->max_pages)
        return fail(FOCR_E_SHAPE, at + "table_stride " + std::to_string(c->table_stride) +
                                      " < max_pages " + std::to_string(c->max_pages));
    if (!c->k || !c->v || (rows && !c->table)) return fail(FOCR_E_ARG, at + "null pointer");
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16)
        return fail(FOCR_E_ARG, at + "k and v pages must be 16-byte aligned");
    out->k = (char *)c->k;
    out->v = (char *)c->v;
    out->table = c->table;
    out->page_stride = (int64_t)(c->page_stride * size);
    out->head_stride = (int64_t)(c->head_stride * size);
    out->table_stride = (int64_t)c->table_stride;
    out->n_pages = (int)c->n_pages;
    out->kv_heads = (int)c->kv_heads;
    out->page_size = (int)c->page_size;
    out->row_bytes = (int)(c->head_dim * size);
    out->max_pages = (int)c->max_pages;
    out->page_div = FastDiv(c->page_size);
    return FOCR_OK;
}

namespace {

// A thread per (token, 16-byte chunk of the token's [kv_heads][head_dim] row)
// of the cache's type, for K and V.  VEC: the source rows are 16-byte aligned.
// Bound by its bytes: 12000 tokens of 8 heads of 128 in bf16, 94 MB, take 14.4 us
// alone (6.5 TB/s) and 17.1 among others; one token of 64 streams 2.1 us, latency.
template <typename S, typename T, bool VEC>
__global__ void __launch_bounds__(256) paged_write_kernel(
    PagedView c, const S *__restrict__ k, const S *__restrict__ v, long long tokens, int rows,
    long long k_stride, long long v_stride, const int32_t *__restrict__ row,
    const int32_t *__restrict__ pos, int chunks_per_head) {
    constexpr int N = 16 / sizeof(T);  // elements of a chunk
    pdl_wait();
    pdl_trigger();
    const int per_token = c.kv_heads * chunks_per_head;
    const long long n = tokens * per_token;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long t = i / per_token;
        const int j = (int)(i - t * per_token);
        const int r = row ? row[t] : (t < rows ? (int)t : -1);
        const int p = pos[t];
        if (r < 0 || r >= rows || p < 0 || p >= c.max_pages * c.page_size) continue;
        const int64_t at = c.offset(c.table + r * c.table_stride, (uint32_t)p);
        if (at < 0) continue;
        const int h = j / chunks_per_head, ch = j - h * chunks_per_head;
        const int64_t dst = at + h * c.head_stride + ch * 16;
#pragma unroll
        for (int which = 0; which < 2; which++) {
            const S *src = (which ? v + t * v_stride : k + t * k_stride) + (int64_t)j * N;
            alignas(16) T y[N];
            if constexpr (sizeof(S) == sizeof(T) && VEC) {
                *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(src);
                if constexpr (!std::is_same<S, T>::value) {
                    float f[N];
                    unpack16<S>(*reinterpret_cast<const uint4 *>(y), f);
#pragma unroll
                    for (int e = 0; e < N; e++) store_f32_as(y, std::is_same<T, __half>::value ? FOCR_F16 : FOCR_BF16, e, f[e]);
                }
            } else {
                float f[N];
                if constexpr (VEC) {
                    constexpr int M = 16 / sizeof(S), C = N > M ? N / M : 1;
                    if constexpr (N >= M) {
#pragma unroll
                        for (int q = 0; q < C; q++)
                            unpack16<S>(reinterpret_cast<const uint4 *>(src)[q], f + q * M);
                    } else {  // 16-bit source into f32 pages: 8 bytes a chunk
                        const uint2 u = *reinterpret_cast<const uint2 *>(src);
                        float g[M];
                        unpack16<S>(make_uint4(u.x, u.y, 0, 0), g);
#pragma unroll
                        for (int e = 0; e < N; e++) f[e] = g[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < N; e++) f[e] = to_f32<S>(src[e]);
                }
#pragma unroll
                for (int e = 0; e < N; e++)
                    store_f32_as(y, sizeof(T) == 4 ? FOCR_F32 : std::is_same<T, __half>::value ? FOCR_F16 : FOCR_BF16, e, f[e]);
            }
            *reinterpret_cast<uint4 *>((which ? c.v : c.k) + dst) = *reinterpret_cast<uint4 *>(y);
        }
    }
}

template <typename S, typename T>
int launch_write(const PagedView &c, size_t rows, const void *k, const void *v, size_t tokens,
                 size_t k_stride, size_t v_stride, const int32_t *row, const int32_t *pos,
                 cudaStream_t st) {
    const int chunks = c.row_bytes / 16;
    const bool vec = ((uintptr_t)k | (uintptr_t)v | (k_stride * sizeof(S)) | (v_stride * sizeof(S))) % 16 == 0;
    const unsigned long long n = (unsigned long long)tokens * c.kv_heads * chunks;
    const unsigned long long want = (n + 255) / 256, most = (unsigned long long)num_sms() * 16;
    const unsigned grid = (unsigned)(want < most ? want : most);
    auto *kernel = vec ? paged_write_kernel<S, T, true> : paged_write_kernel<S, T, false>;
    FOCR_CUDA_TRY(launch_pdl(kernel, grid, 256, 0, st, c, (const S *)k, (const S *)v,
                             (long long)tokens, (int)rows, (long long)k_stride,
                             (long long)v_stride, row, pos, chunks));
    return FOCR_OK;
}

template <typename S>
int write_from(int dtype, const PagedView &c, size_t rows, const void *k, const void *v,
               size_t tokens, size_t k_stride, size_t v_stride, const int32_t *row,
               const int32_t *pos, cudaStream_t st) {
    if (dtype == FOCR_F32)
        return launch_write<S, float>(c, rows, k, v, tokens, k_stride, v_stride, row, pos, st);
    if (dtype == FOCR_F16)
        return launch_write<S, __half>(c, rows, k, v, tokens, k_stride, v_stride, row, pos, st);
    return launch_write<S, __nv_bfloat16>(c, rows, k, v, tokens, k_stride, v_stride, row, pos, st);
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" int focr_paged_write(const focr_paged_cache *cache, const focr_paged_write_args *args, void *stream) {
    return guarded("paged_write", [&]() -> int {
        if (!args) return fail(FOCR_E_ARG, "paged_write: null arguments");
        const void *k = args->k;
        const void *v = args->v;
        const int32_t *row = args->row;
        const int32_t *pos = args->pos;
        const size_t rows = args->rows;
        const size_t tokens = args->tokens;
        const size_t k_stride = args->k_stride;
        const size_t v_stride = args->v_stride;
        const int src_dtype = args->src_dtype;
        PagedView c;
        int rc = paged_view("paged_write", cache, rows, &c);
        if (rc) return rc;
        if (src_dtype != FOCR_F32 && src_dtype != FOCR_F16 && src_dtype != FOCR_BF16)
            return fail(FOCR_E_ARG, "paged_write: unknown source type " + std::to_string(src_dtype));
        if (!tokens || !rows) return FOCR_OK;
        if (!k || !v || !pos) return fail(FOCR_E_ARG, "paged_write: null pointer");
        if (rows > INT32_MAX || tokens > INT32_MAX)
            return fail(FOCR_E_UNSUPPORTED, "paged_write: dimension exceeds int32 range");
        if (!row && tokens > rows)
            return fail(FOCR_E_SHAPE, "paged_write: " + std::to_string(tokens) +
                                          " tokens without rows for a table of " +
                                          std::to_string(rows));
        const size_t wide = (size_t)cache->kv_heads * cache->head_dim;
        if (tokens > 1 && (k_stride < wide || v_stride < wide))
            return fail(FOCR_E_SHAPE, "paged_write: a token stride is shorter than kv_heads * head_dim");
        if (wide > INT32_MAX || k_stride > (size_t)INT64_MAX / 8 / tokens ||
            v_stride > (size_t)INT64_MAX / 8 / tokens)
            return fail(FOCR_E_SHAPE, "paged_write: stride overflow");
        cudaStream_t st = (cudaStream_t)stream;
        if (src_dtype == FOCR_F32)
            return write_from<float>(cache->dtype, c, rows, k, v, tokens, k_stride, v_stride, row, pos, st);
        if (src_dtype == FOCR_F16)
            return write_from<__half>(cache->dtype, c, rows, k, v, tokens, k_stride, v_stride, row, pos, st);
        return write_from<__nv_bfloat16>(cache->dtype, c, rows, k, v, tokens, k_stride, v_stride, row, pos, st);
    });
}
