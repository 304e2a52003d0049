// Attention over a paged cache on the f32 units: any type of query over any type
// of cache.
#pragma once

#include "paged_attention.cuh"

namespace focr {
namespace {

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
    static constexpr int BLOCK = ATTN_WARPS * KEYS;  // positions of a block tile
    static_assert(BLOCK >= 32, "attn_rows counts on it");
    static constexpr int EPL = NC * 16 / (int)sizeof(T);  // dimensions of a lane
};

// Heads that the warps hand over at a time: 2 KB a warp.
template <int D, int GP> constexpr int simt_round() { return GP * D <= 512 ? GP : 512 / D; }
template <typename T, int D, int GP> constexpr int simt_smem() {
    using S = Tile<T, D>;
    static_assert(sizeof(Handover<GP, D>) <= ATTN_WARPS * S::STAGES * 2 * S::HALF, "all heads fit the rings");
    return ATTN_WARPS * S::STAGES * 2 * S::HALF + (int)sizeof(Handover<simt_round<D, GP>(), D>) +
           ATTN_WARPS * GP * S::KEYS * 4 + (ATTN_ROWS + 1) * 4;
}

// The arithmetic runs on the f32 units: with few query heads a kv head the
// loads bound it (a key of 128 16-bit values costs a warp ~25 instructions a
// head against 512 bytes).  16 rows x 8192 positions x 8 kv heads of 128: bf16 92 us
// with one query head (5.8 TB/s), 94 with two; f32 166 us (6.5 TB/s), 178 with four
// query heads, 203 with eight, where 8 warps an SM leave the f32 units waiting, and 402
// with sixteen, in two chunks that each read the cache.
// ALONE: a warp to each (row, head).
template <typename T, int D, int GP, bool ALONE>
__global__ void __launch_bounds__(ATTN_WARPS * 32, 2) paged_attention_kernel(const AttnArgs a) {
    using S = Tile<T, D>;
    constexpr int LPK = S::LPK, KPI = S::KPI, ITS = S::ITS, KEYS = S::KEYS, NC = S::NC, EPL = S::EPL;
    constexpr int EPC = 16 / (int)sizeof(T);  // elements of a chunk
    constexpr int RINGS = ATTN_WARPS * S::STAGES * 2 * S::HALF, HR = simt_round<D, GP>();
    extern __shared__ __align__(128) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    char *ring = smem + warp * S::STAGES * 2 * S::HALF;
    auto &hand = *reinterpret_cast<Handover<HR, D> *>(smem + RINGS);
    float *probs = reinterpret_cast<float *>(smem + RINGS + sizeof(hand)) + warp * GP * KEYS;
    int *pre = reinterpret_cast<int *>(smem + RINGS + sizeof(hand) + ATTN_WARPS * GP * KEYS * 4);
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);

    pdl_wait();
    pdl_trigger();
    if (!ALONE && a.cluster == RUNS) tile_prefix<ATTN_WARPS * 32>(a, pre);

    const int sub = lane / LPK, chunk = lane % LPK;
    // the step whose score this lane holds after the transposing reduction
    const int my_it = (lane & (LPK / 2) ? 4 : 0) + (lane & (LPK / 4) ? 2 : 0) + (lane & (LPK / 8) ? 1 : 0);
    const int my_key = my_it * KPI + sub;

    Run<ALONE> run(a, pre);
    Feed<KEYS, ALONE> feed(run);
    uint32_t bad_stages = 0;   // of the stages in flight, those with a page outside the pool
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
                cp_async16(dst + (it * NC + n) * 512, a.c.k + src, have ? 16 : 0);
                cp_async16(dst + S::HALF + (it * NC + n) * 512, a.c.v + src, have ? 16 : 0);
            }
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
        const int r = sg.r, heads = sg.heads, qh0 = sg.qh0, vis = sg.rv.vis;
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
        bool bad = sg.rv.bad;

        for (int tile = sg.t0; tile < sg.t1; tile++) {
            bad |= bad_stages >> stage & 1;
            bool next_bad;
            const int64_t next = feed.next(a, pre, warp, lane, &next_bad);
            bad_stages = (bad_stages & ~(1u << stage)) | (uint32_t)next_bad << stage;
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
            const int i = first_key<KEYS, ALONE>(tile, warp) + my_key;
            const bool live = i < vis;
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
                if (!live) s[g][0] = -INFINITY;
            }
            // one vote for all heads: their chains run side by side
            bool rises = false;
#pragma unroll
            for (int g = 0; g < GP; g++) rises |= s[g][0] > m[g];
            if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
                for (int g = 0; g < GP; g++) {
                    const float top = fmaxf(m[g], warp_max_f32(s[g][0]));
                    const float f = rescale(m[g], top, a.c2);
                    m[g] = top;
                    l[g] *= f;
#pragma unroll
                    for (int e = 0; e < EPL; e++) acc[g][e] *= f;
                }
            }
#pragma unroll
            for (int g = 0; g < GP; g++) {
                const float p = prob(s[g][0], a.c2, base_of(m[g]));
                l[g] += p;
                probs[g * KEYS + sub * ITS + my_it] = p;
            }
            if (a.scores && live)
#pragma unroll
                for (int g = 0; g < GP; g++)
                    if (g < heads) a.scores[((int64_t)r * a.q_heads + qh0 + g) * a.score_stride + i] = s[g][0];
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

        // the warp's sums over its lanes, then the block's over its warps
        const bool any_bad = __any_sync(0xffffffffu, bad);
#pragma unroll
        for (int g = 0; g < GP; g++) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], o);
            l[g] = any_bad ? NAN : l[g] * (8.0f / LPK);  // LPK / 8 lanes hold the same key
#pragma unroll
            for (int e = 0; e < EPL; e++)
#pragma unroll
                for (int o = LPK; o < 32; o <<= 1) acc[g][e] += __shfl_xor_sync(0xffffffffu, acc[g][e], o);
        }
        if constexpr (ALONE) {
#pragma unroll
            for (int g = 0; g < GP; g++) {
                if (g >= heads) break;
                if (sub == 0)
#pragma unroll
                    for (int e = 0; e < EPL; e += 4) {
                        const int d = (e / EPC * LPK + chunk) * EPC + e % EPC;
                        if (d < a.dim)
                            store4_as(a.out, a.q_type, r * a.out_stride + (long long)(qh0 + g) * a.dim + d,
                                      over4(make_float4(acc[g][e], acc[g][e + 1], acc[g][e + 2], acc[g][e + 3]), l[g], vis));
                    }
                if (a.stat && lane == 0) a.stat[(int64_t)r * a.q_heads + qh0 + g] = make_float2(m[g], 1.0f / l[g]);
            }
            continue;
        }
        auto give = [&](int g, float *o, float *to_m, float *to_l) {
            if (sub == 0)
#pragma unroll
                for (int e = 0; e < EPL; e++) o[(e / EPC * LPK + chunk) * EPC + e % EPC] = acc[g][e];
            if (lane == 0) {
                *to_m = m[g];
                *to_l = l[g];
            }
        };
        if (HR < GP && a.cluster) {   // nothing is to come: all heads at once, where the rings were
            auto &all = *reinterpret_cast<Handover<GP, D> *>(smem);
            cp_async_wait<0>();
            __syncthreads();
#pragma unroll
            for (int g = 0; g < GP; g++) give(g, all.o[warp][g], &all.m[warp][g], &all.l[warp][g]);
            __syncthreads();
            finish_heads<GP, GP, D>(a, sg, all, 0);
            continue;
        }
#pragma unroll
        for (int g0 = 0; g0 < GP; g0 += HR) {
            if (g0 >= heads) break;
#pragma unroll
            for (int i = 0; i < HR; i++) give(g0 + i, hand.o[warp][i], &hand.m[warp][i], &hand.l[warp][i]);
            __syncthreads();
            finish_heads<GP, HR, D>(a, sg, hand, g0);
        }
    }
    cp_async_wait<0>();
}

template <typename T, int D, int GP> int launch_simt(AttnArgs &a, cudaStream_t st) {
    a.gp = GP;
    a.head_chunks = (a.group + GP - 1) / GP;
    a.cluster = cluster_of(a, Tile<T, D>::KEYS);
    a.tile_shift = ilog2(a.cluster == SOLO ? Tile<T, D>::KEYS : Tile<T, D>::BLOCK);
    return launch_attn(a.cluster == SOLO ? paged_attention_kernel<T, D, GP, true> : paged_attention_kernel<T, D, GP, false>,
                       simt_smem<T, D, GP>(), a, st);
}

// 1, 2, 4 or 8 query heads a block: heads that a block does not have cost as much as
// those it has (3 query heads take 4 heads' time), more of them re-read the cache.
template <typename T, int D> int launch_simt_group(AttnArgs &a, cudaStream_t st) {
    if (a.group <= 1) return launch_simt<T, D, 1>(a, st);
    if (a.group <= 2) return launch_simt<T, D, 2>(a, st);
    if (a.group <= 4) return launch_simt<T, D, 4>(a, st);
    return launch_simt<T, D, 8>(a, st);
}
template <typename T> int launch_simt_dim(AttnArgs &a, cudaStream_t st) {
    if (a.dim <= 64) return launch_simt_group<T, 64>(a, st);
    if (a.dim <= 128) return launch_simt_group<T, 128>(a, st);
    return launch_simt_group<T, 256>(a, st);
}

}  // namespace
}  // namespace focr
