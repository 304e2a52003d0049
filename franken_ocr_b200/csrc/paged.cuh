// Shared by the operators on paged K/V caches (paged.cu, paged_attention.cu,
// evict.cu, beam.cu): the cache's view on the device, its checks, and the small
// device helpers they use.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <exception>
#include <string>

#include "common.cuh"

namespace focr {

// Division of n < 2^31 by a divisor fixed at launch: q = (hi(n * mul) + n) >> shift.
struct FastDiv {
    uint32_t mul, shift, d;
    FastDiv() : FastDiv(1) {}
    explicit FastDiv(uint32_t div) : d(div) {
        shift = 0;
        while (((uint64_t)1 << shift) < div) shift++;
        mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - div)) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return (__umulhi(n, mul) + n) >> shift;
    }
};

// A focr_paged_cache as the kernels see it, strides in bytes.
struct PagedView {
    char *k, *v;
    const int32_t *table;
    int64_t page_stride, head_stride, table_stride;  // table_stride in entries
    int n_pages, kv_heads, page_size, row_bytes, max_pages;
    FastDiv page_div;

    // Byte offset of position `pos` of the row whose page list starts at
    // `pages`, without the head's offset; -1 when the page is not in the pool.
    __device__ __forceinline__ int64_t offset(const int32_t *pages, uint32_t pos) const {
        const uint32_t p = page_div.div(pos);
        const int id = pages[p];
        if ((uint32_t)id >= (uint32_t)n_pages) return -1;
        return (int64_t)id * page_stride + (int64_t)(pos - p * (uint32_t)page_size) * row_bytes;
    }
};

inline size_t dtype_bytes(int dtype) { return dtype == FOCR_F32 ? 4 : 2; }

// Checks `c` and fills `*out`; `rows` is the number of table rows the call reads.
int paged_view(const char *ctx, const focr_paged_cache *c, size_t rows, PagedView *out);

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
    return __bfloat162float(x);
}

// The 16 / sizeof(T) values of a 16-byte chunk as f32.
template <typename T> __device__ __forceinline__ void unpack16(const uint4 &u, float *f);
template <> __device__ __forceinline__ void unpack16<float>(const uint4 &u, float *f) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
}
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4 &u, float *f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void unpack16<__half>(const uint4 &u, float *f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

// Element `i` of an array whose type is known at run time only.
__device__ __forceinline__ float load_as_f32(const void *p, int dtype, int64_t i) {
    if (dtype == FOCR_F32) return static_cast<const float *>(p)[i];
    if (dtype == FOCR_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
// One rounding, to nearest even.
__device__ __forceinline__ void store_f32_as(void *p, int dtype, int64_t i, float x) {
    if (dtype == FOCR_F32)
        static_cast<float *>(p)[i] = x;
    else if (dtype == FOCR_F16)
        static_cast<__half *>(p)[i] = __float2half_rn(x);
    else
        static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

__device__ __forceinline__ float warp_max_f32(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Runs the body of a C entry: nothing thrown leaves the library.
template <typename F> int guarded(const char *ctx, F body) {
    try {
        return body();
    } catch (const std::exception &) {
        try {
            return fail(FOCR_E_ALLOC, std::string(ctx) + ": out of host memory");
        } catch (...) {
            return FOCR_E_ALLOC;
        }
    }
}

}  // namespace focr
