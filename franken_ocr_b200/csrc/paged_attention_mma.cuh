// Attention over a paged 16-bit cache on the tensor cores: up to 16 query heads of a
// kv head, of the cache's type or f32, as the rows of a matrix tile.
//
// A warp takes KEYS positions at a time: S = Q K^T and O += P V as 16x8x16 warp
// products straight from the staged rows, whose 16-byte chunks are swizzled by
// the row so that the transposing loads meet no bank twice.  One token's work is
// bound by the cache's bytes, not by the products (48 of them, ~100 cycles of
// an SM, for 8 KB that take ~350 cycles to arrive), so the warp products, which
// leave every warp on its own without a block barrier, cost nothing against
// larger tiles.  P, and a query in f32, are split into parts of the cache's type that
// are multiplied one after the other, so nothing is rounded to fewer bits than the
// output has.
//
// Measured: 8 rows x 131072 positions, 64 / 8 heads of 128, bf16: 645 to 665 us, call
// after call under the power cap 625 to 685 by the GPU, 6.3 to 6.9 TB/s; 16 x 8192 x 8
// heads: 93 us at 3 query heads each, 97 at 8, 99 at 16 (5.4 TB/s).
#pragma once

#include "paged_attention.cuh"

namespace focr {
namespace {

template <int D> struct MmaTile {
    static constexpr int DB = D * 2;
    static constexpr int CH = DB / 16;
    static constexpr int KEYS = D == 64 ? 32 : 16;
    static constexpr int HALF = KEYS * DB;
    static constexpr int STAGES = HALF > 4096 ? 2 : 3;
    static constexpr int BLOCK = ATTN_WARPS * KEYS;
    static_assert(BLOCK >= 32, "attn_rows counts on it");
};
// Heads that the warps hand over at a time: 2 KB a warp, or all where one block
// fills an SM.
template <int D> constexpr int mma_round() { return D == 256 ? 16 : 512 / D; }
// At head_dim 256 the query's registers are needed elsewhere: it lies in shared
// memory, swizzled like the rows.
template <int D> constexpr int mma_q_bytes() { return D == 256 ? 16 * D * 2 : 0; }
template <int D> constexpr int mma_smem() {
    return ATTN_WARPS * MmaTile<D>::STAGES * 2 * MmaTile<D>::HALF + (int)sizeof(Handover<mma_round<D>(), D>) +
           mma_q_bytes<D>() + (ATTN_ROWS + 1) * 4;
}

// c += a b.  The addend has registers of its own, so that zeros need none.
template <typename T> __device__ __forceinline__ void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    float d[4];
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    c[0] = d[0];
    c[1] = d[1];
    c[2] = d[2];
    c[3] = d[3];
}
template <bool TRANS> __device__ __forceinline__ void ldmatrix4(uint32_t *r, uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Two f32 additions at a time.
__device__ __forceinline__ void add_pair(float *a, const float *b) {
    asm("{.reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;}"
        : "+f"(a[0]), "+f"(a[1]) : "f"(b[0]), "f"(b[1]));
}
// The pair (x, y) in T, and in *x, *y what it leaves of them.
template <typename T> __device__ __forceinline__ uint32_t take_pair(float *x, float *y) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(*x, *y);
        const float2 f = __half22float2(h);
        *x -= f.x;
        *y -= f.y;
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(*x, *y);
        const float2 f = __bfloat1622float2(h);
        *x -= f.x;
        *y -= f.y;
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// A pair of probabilities in N parts of T, whose sum they are.  Each part of one above 0
// is above 0 too, as an infinite value times a negative part, or 0, would make NaN of it;
// those of 0 are 0.  So all parts but the last are cut off, and a lower one has 2^-30 of
// the probability added, or, in f16, which reaches no further down, is 2^-24 at least.
template <typename T, int N> __device__ __forceinline__ void split_probs(float x, float y, uint32_t (*to)[4], int at) {
    if constexpr (std::is_same<T, __half>::value) {
        const float fx = fminf(x * 0x1p127f, 0x1p-24f), fy = fminf(y * 0x1p127f, 0x1p-24f);   // 0 for 0
#pragma unroll
        for (int p = 0; p < N; p++) {
            x = fmaxf(x, fx);
            y = fmaxf(y, fy);
            if (p == N - 1) {
                to[p][at] = take_pair<T>(&x, &y);
            } else {
                asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(to[p][at]) : "f"(y), "f"(x));
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&to[p][at]));
                x -= f.x;
                y -= f.y;
            }
        }
    } else {   // an f32's upper half is it cut off to bf16
        const float x0 = x, y0 = y;
#pragma unroll
        for (int p = 0; p < N; p++) {
            if (p == N - 1) {
                to[p][at] = take_pair<T>(&x, &y);
            } else {
                const uint32_t bx = __float_as_uint(x), by = __float_as_uint(y);
                to[p][at] = __byte_perm(bx, by, 0x7632);
                x = __fmaf_rn(x0, 0x1p-30f, x - __uint_as_float(bx & 0xffff0000u));
                y = __fmaf_rn(y0, 0x1p-30f, y - __uint_as_float(by & 0xffff0000u));
            }
        }
    }
}

// PARTS: how many values of T a query element and a probability are split into.
// A query of type T is one, and its probabilities two (16 bits of bf16, 22 of f16, the
// last rounded); an f32 query takes three of both (24 bits of bf16, 33 of f16).
// ALONE: a warp to each (row, head).
template <typename T, int D, bool F32Q, bool ALONE>
__global__ void __launch_bounds__(ATTN_WARPS * 32, D == 256 ? 1 : 2) paged_attention_mma_kernel(const AttnArgs a) {
    using S = MmaTile<D>;
    constexpr int GP = 16, KEYS = S::KEYS, NT = KEYS / 8, ITS = S::HALF / 512, HR = mma_round<D>();
    constexpr int QP = F32Q ? 3 : 1, PP = F32Q ? 3 : 2;
    constexpr bool QS = mma_q_bytes<D>() > 0;
    static_assert(!(QS && F32Q), "an f32 query's parts are kept in registers");
    constexpr bool HALF = std::is_same<T, __half>::value;
    // f16 holds nothing below 2^-24: probabilities, at most 1, are scaled up, and a
    // head's f32 query by the power of two that brings its largest value near 2^14
    constexpr float PS = HALF ? 16384.0f : 1.0f;
    constexpr int RINGS = ATTN_WARPS * S::STAGES * 2 * S::HALF;
    static_assert(sizeof(Handover<GP, D>) <= RINGS, "all heads fit the rings");
    extern __shared__ __align__(128) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    char *ring = smem + warp * S::STAGES * 2 * S::HALF;
    auto &hand = *reinterpret_cast<Handover<HR, D> *>(smem + RINGS);
    char *qs = smem + RINGS + sizeof(hand);
    int *pre = reinterpret_cast<int *>(qs + mma_q_bytes<D>());
    const uint32_t qs_s = (uint32_t)__cvta_generic_to_shared(qs);
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);

    pdl_wait();
    pdl_trigger();
    if (!ALONE && a.cluster == RUNS) tile_prefix<ATTN_WARPS * 32>(a, pre);

    const int qr = lane >> 2, qc = (lane & 3) * 2;   // this lane's row and columns of a tile
    const int mi = lane >> 3, rr = lane & 7;         // its matrix and row when loading one
    Run<ALONE> run(a, pre);
    Feed<KEYS, ALONE> feed(run);
    uint32_t bad_stages = 0;   // of the stages in flight, those with a page outside the pool
    auto issue = [&](int stage, int64_t mine) {
        const uint32_t dst = ring_s + stage * 2 * S::HALF;
#pragma unroll
        for (int it = 0; it < ITS; it++) {
            const int x = it * 32 + lane, key = x / S::CH, c = x % S::CH;
            const int64_t o = __shfl_sync(0xffffffffu, mine, key);
            const bool have = o >= 0 && c * 16 < a.c.row_bytes;
            const int64_t src = have ? o + c * 16 : 0;
            const uint32_t to = dst + key * S::DB + ((c ^ (key & 7)) << 4);
            cp_async16(to, a.c.k + src, have ? 16 : 0);
            cp_async16(to + S::HALF, a.c.v + src, have ? 16 : 0);
        }
    };
#pragma unroll
    for (int s = 0; s < S::STAGES; s++) {
        bool bad;
        issue(s, feed.next(a, pre, warp, lane, &bad));
        bad_stages |= (uint32_t)bad << s;
        cp_async_commit();
    }
    if constexpr (!ALONE) finish_empty_rows(a, pre);

    int stage = 0;
    Segment sg;
    while (run.next(a, pre, &sg)) {
        const int r = sg.r, heads = sg.heads, vis = sg.rv.vis;
        uint32_t qa[QP][QS ? 1 : D / 16][4];
        float unscale[2] = {1.0f, 1.0f};
        if constexpr (F32Q) {
            const float *qp = static_cast<const float *>(a.q) + r * a.q_stride + (long long)sg.qh0 * a.dim;
            float qf[D / 16][4][2], scale[2] = {1.0f, 1.0f};
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int g = qr + (x & 1) * 8, d = ks * 16 + (x >> 1) * 8 + qc;
                    const bool have = g < heads && d < a.dim;   // dim is even
                    qf[ks][x][0] = have ? qp[g * a.dim + d] : 0.0f;
                    qf[ks][x][1] = have ? qp[g * a.dim + d + 1] : 0.0f;
                }
            if constexpr (HALF) {
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    float top = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                        for (int x = y; x < 4; x += 2) top = fmaxf(top, fmaxf(fabsf(qf[ks][x][0]), fabsf(qf[ks][x][1])));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // 2^(13 - exponent), between 2^-100 and 2^100; 0, inf and NaN as they are
                    const int e = (int)(__float_as_uint(top) >> 23) - 127;
                    if (top > 0.0f && e < 128) {
                        const int up = max(-100, min(100, 13 - e));
                        scale[y] = __int_as_float((127 + up) << 23);
                        unscale[y] = __int_as_float((127 - up) << 23);
                    }
                }
            }
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    float q0 = qf[ks][x][0] * scale[x & 1], q1 = qf[ks][x][1] * scale[x & 1];
#pragma unroll
                    for (int p = 0; p < QP; p++) qa[p][ks][x] = take_pair<T>(&q0, &q1);
                }
        } else if constexpr (QS) {
            const uint16_t *qp = static_cast<const uint16_t *>(a.q) + r * a.q_stride + (long long)sg.qh0 * a.dim;
            for (int x = threadIdx.x; x < GP * D; x += ATTN_WARPS * 32) {   // the block is past its last use
                const int g = x / D, d = x % D;
                *reinterpret_cast<uint16_t *>(qs + g * S::DB + ((d / 8 ^ (g & 7)) << 4) + d % 8 * 2) =
                    g < heads && d < a.dim ? qp[g * a.dim + d] : (uint16_t)0;
            }
            __syncthreads();
        } else {
            const uint16_t *qp = static_cast<const uint16_t *>(a.q) + r * a.q_stride + (long long)sg.qh0 * a.dim;
            const bool pairs = (uintptr_t)qp % 4 == 0;   // dim is even
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int g = qr + (x & 1) * 8, d = ks * 16 + (x >> 1) * 8 + qc;
                    const uint16_t *p = qp + g * a.dim + d;
                    qa[0][ks][x] = 0;
                    if (g < heads && d < a.dim)
                        qa[0][ks][x] = pairs ? *reinterpret_cast<const uint32_t *>(p) : p[0] | (uint32_t)p[1] << 16;
                }
        }
        float acc[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < D / 8; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
        bool bad = sg.rv.bad;

        for (int tile = sg.t0; tile < sg.t1; tile++) {
            bad |= bad_stages >> stage & 1;
            bool next_bad;
            const int64_t next = feed.next(a, pre, warp, lane, &next_bad);
            bad_stages = (bad_stages & ~(1u << stage)) | (uint32_t)next_bad << stage;
            cp_async_wait<S::STAGES - 1>();
            __syncwarp();
            const uint32_t ks_s = ring_s + stage * 2 * S::HALF, vs_s = ks_s + S::HALF;
            // The tensor cores cut their sums off where f32 would round, always
            // towards zero, so a long chain is off by a share that grows with its
            // length (P V in one chain over 2^20 positions: 2^-9 of the output).  A
            // chain of P V therefore ends with its tile and is joined by f32 additions;
            // a score's is head_dim / 16 steps, of which an f32 query takes every other.
            constexpr int CHAINS = F32Q ? 3 : 1;   // even steps, odd steps, the query's lower parts
            float s[NT][4], sc[CHAINS][NT][4];
#pragma unroll
            for (int c = 0; c < CHAINS; c++)
#pragma unroll
                for (int t = 0; t < NT; t++) sc[c][t][0] = sc[c][t][1] = sc[c][t][2] = sc[c][t][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                if constexpr (QS) ldmatrix4<false>(qa[0][0], qs_s + ((mi & 1) * 8 + rr) * S::DB + (((ks * 2 + (mi >> 1)) ^ rr) << 4));
#pragma unroll
                for (int p = 0; p < KEYS / 16; p++) {
                    uint32_t b[4];
                    ldmatrix4<false>(b, ks_s + (p * 16 + (mi >> 1) * 8 + rr) * S::DB + (((ks * 2 + (mi & 1)) ^ rr) << 4));
#pragma unroll
                    for (int part = QP - 1; part >= 0; part--) {
                        auto &to = sc[F32Q ? (part ? 2 : ks & 1) : 0];
                        mma16816<T>(to[2 * p], qa[part][QS ? 0 : ks], b[0], b[1]);
                        mma16816<T>(to[2 * p + 1], qa[part][QS ? 0 : ks], b[2], b[3]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    s[t][x] = sc[0][t][x];
                    if constexpr (F32Q) {
                        // an infinite score is that of the query's upper part: the lower
                        // ones have either sign, or are 0
                        s[t][x] += sc[CHAINS / 2][t][x];
                        if (fabsf(s[t][x]) != INFINITY) s[t][x] += sc[CHAINS - 1][t][x];
                    }
                }
            if constexpr (F32Q && HALF)
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[t][x] *= unscale[x >> 1];
            const int i0 = first_key<KEYS, ALONE>(tile, warp) + qc;
            if (a.scores) {   // pairs: the stride is even, what lies behind vis is never read
                float *sp = a.scores + ((int64_t)r * a.q_heads + sg.qh0 + qr) * a.score_stride + i0;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (i0 + t * 8 >= vis) break;
                    if (qr < heads) *reinterpret_cast<float2 *>(sp + t * 8) = make_float2(s[t][0], s[t][1]);
                    if (qr + 8 < heads)
                        *reinterpret_cast<float2 *>(sp + 8ll * a.score_stride + t * 8) = make_float2(s[t][2], s[t][3]);
                }
            }
            float top[2] = {-INFINITY, -INFINITY};
            if (i0 - qc + KEYS > vis)   // the row's last tile
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (i0 + t * 8 + (x & 1) >= vis) s[t][x] = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int x = 0; x < 4; x++) top[x >> 1] = fmaxf(top[x >> 1], s[t][x]);
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    float n = fmaxf(m[y], top[y]);
                    n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 1));
                    n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 2));
                    const float f = rescale(m[y], n, a.c2);
                    m[y] = n;
                    l[y] *= f;
#pragma unroll
                    for (int j = 0; j < D / 8; j++) {
                        acc[j][2 * y] *= f;
                        acc[j][2 * y + 1] *= f;
                    }
                }
            }
            const float base[2] = {base_of(m[0]), base_of(m[1])};
            uint32_t pa[KEYS / 16][PP][4];
#pragma unroll
            for (int kk = 0; kk < KEYS / 16; kk++)
#pragma unroll
                for (int x = 0; x < 4; x++) {  // registers: (row, low keys), (row + 8, low), (row, high), (row + 8, high)
                    const int t = 2 * kk + (x >> 1), y = x & 1;
                    float p0 = prob(s[t][2 * y], a.c2, base[y]) * PS, p1 = prob(s[t][2 * y + 1], a.c2, base[y]) * PS;
                    l[y] += p0 + p1;
                    split_probs<T, PP>(p0, p1, pa[kk], x);
                }
#pragma unroll
            for (int jp = 0; jp < D / 16; jp++) {
                float short_sum[2][4] = {};
#pragma unroll
                for (int kk = 0; kk < KEYS / 16; kk++) {
                    uint32_t b[4];
                    ldmatrix4<true>(b, vs_s + (kk * 16 + (mi & 1) * 8 + rr) * S::DB + (((jp * 2 + (mi >> 1)) ^ rr) << 4));
#pragma unroll
                    for (int p = PP - 1; p >= 0; p--) {
                        mma16816<T>(short_sum[0], pa[kk][p], b[0], b[1]);
                        mma16816<T>(short_sum[1], pa[kk][p], b[2], b[3]);
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; x += 2) {
                    add_pair(&acc[2 * jp][x], &short_sum[0][x]);
                    add_pair(&acc[2 * jp + 1][x], &short_sum[1][x]);
                }
            }
            __syncwarp();
            issue(stage, next);
            cp_async_commit();
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        }

        const bool any_bad = __any_sync(0xffffffffu, bad);
#pragma unroll
        for (int y = 0; y < 2; y++) {
            l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
            l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
            l[y] = any_bad ? NAN : l[y] * (1.0f / PS);
        }
        if constexpr (ALONE) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int g = qr + y * 8;
                if (g >= heads) break;
                const float by = 1.0f / PS, L = !vis && l[y] == 0.0f ? 1.0f : l[y];   // as over4
                const int64_t to = r * a.out_stride + (long long)(sg.qh0 + g) * a.dim + qc;
#pragma unroll
                for (int j = 0; j < D / 8; j++)
                    if (j * 8 < a.dim) store2_as(a.out, a.q_type, to + j * 8, acc[j][2 * y] * by / L, acc[j][2 * y + 1] * by / L);
                if (a.stat && (lane & 3) == 0) a.stat[(int64_t)r * a.q_heads + sg.qh0 + g] = make_float2(m[y], 1.0f / l[y]);
            }
            continue;
        }
        auto give = [&](int y, float *o, float *to_m, float *to_l) {
#pragma unroll
            for (int j = 0; j < D / 8; j++)
                *reinterpret_cast<float2 *>(o + j * 8 + qc) =
                    make_float2(acc[j][2 * y] * (1.0f / PS), acc[j][2 * y + 1] * (1.0f / PS));
            if ((lane & 3) == 0) {
                *to_m = m[y];
                *to_l = l[y];
            }
        };
        if (HR < GP && a.cluster) {   // nothing is to come: all heads at once, where the rings were
            auto &all = *reinterpret_cast<Handover<GP, D> *>(smem);
            cp_async_wait<0>();
            __syncthreads();
#pragma unroll
            for (int y = 0; y < 2; y++) give(y, all.o[warp][qr + y * 8], &all.m[warp][qr + y * 8], &all.l[warp][qr + y * 8]);
            __syncthreads();
            finish_heads<GP, GP, D>(a, sg, all, 0);
            continue;
        }
#pragma unroll
        for (int g0 = 0; g0 < GP; g0 += HR) {
            if (g0 >= heads) break;
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int i = qr + y * 8 - g0;
                if (i >= 0 && i < HR) give(y, hand.o[warp][i], &hand.m[warp][i], &hand.l[warp][i]);
            }
            __syncthreads();
            finish_heads<GP, HR, D>(a, sg, hand, g0);
        }
    }
    cp_async_wait<0>();
}

template <typename T, int D, bool F32Q> int launch_mma(AttnArgs &a, cudaStream_t st) {
    a.gp = 16;
    a.head_chunks = (a.group + 15) / 16;
    constexpr bool WARPS = mma_q_bytes<D>() == 0;   // a query in shared memory is the block's
    a.cluster = cluster_of(a, WARPS ? MmaTile<D>::KEYS : 0);
    a.tile_shift = ilog2(a.cluster == SOLO ? MmaTile<D>::KEYS : MmaTile<D>::BLOCK);
    return launch_attn(a.cluster == SOLO ? paged_attention_mma_kernel<T, D, F32Q, WARPS> : paged_attention_mma_kernel<T, D, F32Q, false>,
                       mma_smem<D>(), a, st);
}
// Whether this kernel takes the call.  16 rows x 8192 positions x 8 kv heads, bf16, this
// kernel against the f32 units:
//   query of the cache's type, from 3 query heads a kv head on: head_dim 64: 2 heads
//   47.2 / 52.5 us, 3 heads 47.0 / 60.3; 128: 94.1 / 92.8, 93.0 / 102.7; 256: 179 / 176,
//   186 / 191, 6 heads 187 / 317;
//   f32 query, three times the products and short chains, from 5 heads on: head_dim 64:
//   4 heads 59.2 / 58.0, 5 heads 59.4 / 98.9; 128: 4 heads 107 / 101, 5 heads 110 / 172;
//   not at 256, where its parts do not fit the registers.
template <typename T> bool mma_takes(const AttnArgs &a) {
    constexpr int own = std::is_same<T, __half>::value ? FOCR_F16 : FOCR_BF16;
    if (a.q_type == own) return a.group >= 3;
    return a.q_type == FOCR_F32 && a.dim <= 128 && a.group >= 5;
}
template <typename T> int launch_mma_dim(AttnArgs &a, cudaStream_t st) {
    if (a.q_type == FOCR_F32)
        return a.dim <= 64 ? launch_mma<T, 64, true>(a, st) : launch_mma<T, 128, true>(a, st);
    if (a.dim <= 64) return launch_mma<T, 64, false>(a, st);
    if (a.dim <= 128) return launch_mma<T, 128, false>(a, st);
    return launch_mma<T, 256, false>(a, st);
}

}  // namespace
}  // namespace focr
