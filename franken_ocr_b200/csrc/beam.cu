// Beam search over the decoder's logits: the choice of the next beams
// (focr_beam_select) and the reordering of their pages (focr_beam_reorder).
//
// A candidate (beam i, token t) scores
//   cum_i + ((x_t - m_i) - log sum_u exp(x_u - m_i)),   m_i = max_u x_u,
// and candidates are ranked by score, then lower beam, then larger logit, then
// lower token.  The scores are held in 64 bits, and a sum is good to 2^-27 of itself
// (equal rows have equal ones): candidates of different beams often lie closer than f32
// resolves, and a choice, unlike a value, cannot be a little off.
//
// Within one beam the ranking is the logits' own, so no sum is needed to
// shorten the list: select_part_kernel reads each vocabulary strip once and
// keeps its sum and its n largest logits; select_join_kernel, a block per
// entry, has beams * strips * n candidates left to rank.
#include "paged.cuh"

namespace focr {
namespace {

constexpr int ST = 256;    // threads of both kernels
constexpr int MAX_N = 64;
constexpr int LIST = 1024; // candidates ranked together

struct SelectArgs {
    const void *x;
    const float *cum;
    const uint8_t *done;
    float *score_out;
    int32_t *parent_out, *token_out;
    long long row_stride;            // elements between the logits of two beams
    int beams, vocab, n, strips, end_token;
    FastDiv by_n, by_strips;
    // workspace, per (row, strip): n (logit, token) pairs, (max, sum)
    float *cx;
    int32_t *ct;
    float *pm;
    double *ps;
};

// Threads of a group: 4 groups for each of n choices, 32 at least and 256 at most.
__device__ __forceinline__ int group_lanes(int n) { return n <= 8 ? 8 : n <= 16 ? 4 : n <= 32 ? 2 : 1; }

__device__ __forceinline__ float block_max_f32(float v, float *sh) {
    v = warp_max_f32(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = sh[0];
#pragma unroll
    for (int w = 1; w < ST / 32; w++) m = fmaxf(m, sh[w]);
    return m;
}

constexpr float LARGEST = 3.402823466e38f;
constexpr float SHIFT = 786432.0f;   // 1.5 * 2^19: adding it rounds to sixteenths in the low bits

// Two f32 operations at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{.reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
        " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
        " mov.b64 {%0, %1}, d;}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n"
        " mov.b64 {%0, %1}, d;}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// 2^(i / 16), as the bits of a double.
__constant__ unsigned long long POWER[16] = {
    0x3ff0000000000000ull, 0x3ff0b5586cf9890full, 0x3ff172b83c7d517bull, 0x3ff2387a6e756238ull,
    0x3ff306fe0a31b715ull, 0x3ff3dea64c123422ull, 0x3ff4bfdad5362a27ull, 0x3ff5ab07dd485429ull,
    0x3ff6a09e667f3bcdull, 0x3ff7a11473eb0187ull, 0x3ff8ace5422aa0dbull, 0x3ff9c49182a3f090ull,
    0x3ffae89f995ad3adull, 0x3ffc199bdd85529cull, 0x3ffd5818dcfba487ull, 0x3ffea4afa2a490daull};

// Adds 2^(x log2 e - base) of four x between (base - 100) / log2 e and (base + 1) / log2 e
// to *sum, each to 2^-27 of itself.  With n / 16 the nearest sixteenth to x log2 e, the
// value is 2^(n / 16) (1 + p), p = 2^s - 1 with |s| <= 1/32 and |p| < 2^-5.5: the first
// factor comes from a table and is summed in 64 bits; what is rounded to f32 lies 2^-5
// below it.  s: two roundings of 2^-30; p: two of 2^-30; the four's sum: three of 2^-30.5;
// together 2^-27.5.  log2 e is in two parts (Cody and Waite).
// power: the table in shared memory, 16 entries over 32 banks, less i << 48, which the
// shifted index adds again.
__device__ __forceinline__ void add_exp4(float2 xa, float2 xb, float base, const uint2 *power, double *sum) {
    const float up = SHIFT - base;   // base is an integer: exact
    float2 rest = both(0.0f);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float2 x = i ? xb : xa;
        const float2 t = fma2(x, both(1.44269502f), both(up));
        const uint32_t t0 = __float_as_uint(t.x), t1 = __float_as_uint(t.y);   // low bits: n - 16 base
        const float2 n = fma2(t, both(-1.0f), both(up));                       // -n / 16
        const float2 s = fma2(x, both(1.92596299e-8f), fma2(x, both(1.44269502f), n));
        float2 p = fma2(s, both(9.61812911e-3f), both(5.55041087e-2f));        // ln 2^k / k!
        p = fma2(p, s, both(2.40226507e-1f));
        p = fma2(p, s, both(6.93147181e-1f));
        p = mul2(p, s);
        const uint2 w0 = power[t0 & 15], w1 = power[t1 & 15];
        const uint32_t h0 = (t0 << 16) + w0.y, h1 = (t1 << 16) + w1.y;
        *sum += __hiloint2double((int)h0, (int)w0.x);
        *sum += __hiloint2double((int)h1, (int)w1.x);
        // the same as f32: 8 bits of exponent, its bias 896 less, and 23 of the fraction
        const float2 f = make_float2(__uint_as_float(__funnelshift_l(w0.x, h0, 3) + 0x40000000u),
                                     __uint_as_float(__funnelshift_l(w1.x, h1, 3) + 0x40000000u));
        rest = fma2(p, f, rest);
    }
    *sum += rest.x + rest.y;
}

// One strip of one row's logits, held in registers (PER a thread, read once, 16
// bytes at a time where the row begins on such a boundary): its largest logit,
// its sum of exponentials and its n largest candidates.  A thread's logits do
// not depend on the row's alignment, so equal rows give equal sums.
//
// The sum: every term to 2^-27 of itself (add_exp4), summed in 64 bits, so that equal
// logits, whose errors all fall to one side, leave less than 2^-27 of it too (3e-9
// measured; terms of 24 bits, summed in fours as f32, 1.1e-7 and 7 us less for 32 x 8
// rows of 129280 logits).  The largest logits count 1 each, exactly: rows that leave one
// token, or equal ones, tie where their beams do.  The 64-bit exponential of every logit
// would cost several times the strip's load.
//
// The n largest: at least n logits reach the n-th largest of the maxima of 2n or
// more groups of threads, and hardly more do; these are collected and ranked by
// counting.
// Where too many reach it (a constant row), the n are taken one by one.
//
// Bound by instructions, half of them the exponentials, and by the three barriers of a
// short block: 32 x 8 rows of 129280 f32 logits, 132 MB, take 56 us with the join behind
// them, 2.4 TB/s.
template <typename T, int PER>
__global__ void __launch_bounds__(ST, 4) select_part_kernel(const SelectArgs a) {
    constexpr int V = 16 / (int)sizeof(T), STRIP = ST * PER;
    __shared__ __align__(16) float tops[ST];
    __shared__ float sh[ST / 32], lx[LIST];
    __shared__ int lt[LIST], count;
    __shared__ float bound;
    __shared__ double shd[ST / 32];
    __shared__ int shc[ST / 32];
    __shared__ __align__(8) uint2 power[16];
    const int strip = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    if (t < 16) power[t] = make_uint2((uint32_t)POWER[t], (uint32_t)(POWER[t] >> 32) - ((uint32_t)t << 16));
    pdl_wait();
    pdl_trigger();
    const T *x = static_cast<const T *>(a.x) + row * a.row_stride;
    const bool vec = (uintptr_t)x % 16 == 0;
    const int first = strip * STRIP;
    float v[PER];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER / V; i++) {
        const int c = first + (i * ST + t) * V;
        if (vec && c + V <= a.vocab) {
            unpack16<T>(*reinterpret_cast<const uint4 *>(x + c), v + i * V);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++)
                v[i * V + e] = c + e < a.vocab ? to_f32<T>(x[c + e]) : -INFINITY;
        }
    }
    auto token = [&](int i) { return first + (i / V * ST + t) * V + i % V; };
    // NaN loses every maximum and comparison; +inf counts as the largest number
    float most[PER / 4];   // of each four
#pragma unroll
    for (int g = 0; g < PER / 4; g++) {
        most[g] = fmaxf(fmaxf(v[4 * g], v[4 * g + 1]), fmaxf(v[4 * g + 2], v[4 * g + 3]));
        top = fmaxf(top, most[g]);
    }
    if (top == INFINITY) {
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = v[i] == INFINITY ? LARGEST : v[i];
#pragma unroll
        for (int g = 0; g < PER / 4; g++) most[g] = fminf(most[g], LARGEST);
        top = LARGEST;
    }
    const int lanes = group_lanes(a.n), groups = ST / lanes;
    for (int o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (t % lanes == 0) tops[t / lanes] = top;
    if (t == 0) {
        count = 0;
        bound = -INFINITY;
    }
    const float m = block_max_f32(top, sh);
    const long long at = (long long)row * a.strips + strip;
    if (m == -INFINITY) {
        for (int k = t; k < a.n; k += ST) a.ct[at * a.n + k] = -1;
        if (t == 0) {
            a.pm[at] = m;
            a.ps[at] = 0.0;
        }
        return;
    }
    if (t < groups) {  // the group whose maximum ranks n-th names the bound
        const float mine = tops[t];
        int rank = 0;
        for (int j = 0; j < groups; j += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(tops + j);
            rank += (o.x > mine || (o.x == mine && j < t)) + (o.y > mine || (o.y == mine && j + 1 < t)) +
                    (o.z > mine || (o.z == mine && j + 2 < t)) + (o.w > mine || (o.w == mine && j + 3 < t));
        }
        if (rank == a.n - 1) bound = mine;
    }
    // far from 0 the differences to the maximum are exact and stay small
    const float zero = fabsf(m) >= 1024.0f ? m : 0.0f, high = m - zero;
    const float base = rintf(__fmul_rn(high, 1.44269502f)), none = high - 65.0f;   // e^-65 of the largest adds nothing
    const float2 minus = both(-zero);
    double sum = 0.0;
    int ones = 0;
#pragma unroll
    for (int g = 0; g < PER / 4; g++) {
        float2 y0 = add2(make_float2(v[4 * g], v[4 * g + 1]), minus), y1 = add2(make_float2(v[4 * g + 2], v[4 * g + 3]), minus);
        y0 = make_float2(fmaxf(y0.x, none), fmaxf(y0.y, none));   // NaN too
        y1 = make_float2(fmaxf(y1.x, none), fmaxf(y1.y, none));
        if (most[g] == m) {   // rarely
            if (v[4 * g] == m) ones++, y0.x = none;
            if (v[4 * g + 1] == m) ones++, y0.y = none;
            if (v[4 * g + 2] == m) ones++, y1.x = none;
            if (v[4 * g + 3] == m) ones++, y1.y = none;
        }
        add_exp4(y0, y1, base, power, &sum);
    }
    __syncthreads();
    // the candidates
    const float low = bound;
    int c = 0;
#pragma unroll
    for (int g = 0; g < PER / 4; g++)
        if (most[g] >= low)
#pragma unroll
            for (int i = 4 * g; i < 4 * g + 4; i++) c += v[i] >= low && v[i] > -INFINITY;
    if (c) {
        int k = atomicAdd(&count, c);
        if (k + c <= LIST)
#pragma unroll
            for (int g = 0; g < PER / 4; g++)
                if (most[g] >= low)
#pragma unroll
                    for (int i = 4 * g; i < 4 * g + 4; i++)
                        if (v[i] >= low && v[i] > -INFINITY) {
                            lx[k] = v[i];
                            lt[k++] = token(i);
                        }
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    ones = __reduce_add_sync(0xffffffffu, ones);
    if ((t & 31) == 0) {
        shd[t >> 5] = sum;
        shc[t >> 5] = ones;
    }
    __syncthreads();
    const int got = count;
    const bool listed = got <= LIST;
    if (listed && t >= 32) {   // ranked by the other warps, while the first one sums up
        for (int i = t - 32; i < got; i += ST - 32) {
            const float y = lx[i];
            const int c = lt[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < got; j++) rank += (lx[j] > y) | ((lx[j] == y) & (lt[j] < c));
            if (rank < a.n) {
                a.cx[at * a.n + rank] = y;
                a.ct[at * a.n + rank] = c;
            }
        }
        for (int k = got + t - 32; k < a.n; k += ST - 32) a.ct[at * a.n + k] = -1;   // fewer than n: all are listed
        return;
    }
    if (t == 0) {
        for (int w = 1; w < ST / 32; w++) {
            sum += shd[w];
            ones += shc[w];
        }
        a.pm[at] = m;
        // the other terms were taken relative to 2^base
        a.ps[at] = ones + sum * exp((double)base * 0.693147180559945309 - (double)high);
    }
    if (listed) return;
    float last = INFINITY;
    int last_token = -1;
    for (int k = 0; k < a.n; k++) {  // LIST > n: there are that many
        float y = -INFINITY;
        int c = INT_MAX;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (v[i] < last || (v[i] == last && token(i) > last_token))
                if (v[i] > y || (v[i] == y && token(i) < c)) {
                    y = v[i];
                    c = token(i);
                }
        for (int o = 16; o > 0; o >>= 1) {
            const float oy = __shfl_xor_sync(0xffffffffu, y, o);
            const int oc = __shfl_xor_sync(0xffffffffu, c, o);
            if (oy > y || (oy == y && oc < c)) {
                y = oy;
                c = oc;
            }
        }
        __syncthreads();
        if ((t & 31) == 0) {
            lx[t >> 5] = y;
            lt[t >> 5] = c;
        }
        __syncthreads();
        last = lx[0];
        last_token = lt[0];
        for (int w = 1; w < ST / 32; w++)
            if (lx[w] > last || (lx[w] == last && lt[w] < last_token)) {
                last = lx[w];
                last_token = lt[w];
            }
        if (t == 0) {
            a.cx[at * a.n + k] = last;
            a.ct[at * a.n + k] = last_token;
        }
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
__device__ __forceinline__ Cand no_cand() { return Cand{-INFINITY, -INFINITY, INT_MAX, INT_MAX}; }

// A block per entry: the rows' sums, then the n best of all strips' candidates.
// The n-th best score among the strips' first candidates (a thread takes the best
// of those it sees), or among all where the strips are few, bounds the others; what
// reaches it is ranked by counting.
// Latency bounds it: 3 us for 1 x 4 beams, 3 to 4 for 32 x 8.
__global__ void __launch_bounds__(ST) select_join_kernel(const SelectArgs a) {
    __shared__ double row_m[MAX_N], row_s[MAX_N];
    __shared__ float row_cum[MAX_N];
    __shared__ uint8_t row_done[MAX_N];
    __shared__ __align__(16) char list_mem[LIST * sizeof(Cand)];
    __shared__ __align__(16) double heads[ST], tops[ST], list_score[LIST];
    __shared__ double bound;
    __shared__ int count;
    Cand *list = reinterpret_cast<Cand *>(list_mem);
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lists = a.beams * a.strips;
    const long long at = (long long)b * lists * a.n;
    // the thread's first candidates are on their way while the sums are formed
    constexpr int U = 4;
    float head_x = 0.0f, early_x[U];
    int head_t = -1, early_t[U];
    if (t < lists) {
        head_x = a.cx[at + (long long)t * a.n];
        head_t = a.ct[at + (long long)t * a.n];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int j = t + u * ST;
        early_x[u] = j < lists * a.n ? a.cx[at + j] : 0.0f;
        early_t[u] = j < lists * a.n ? a.ct[at + j] : -1;
    }
    for (int i = warp; i < a.beams; i += ST / 32) {
        const long long row = (long long)b * a.beams + i;
        const float cum = a.cum[row];
        const uint8_t done = a.done ? a.done[row] : 0;
        float m = -INFINITY, m2[2];
        double s2[2], sum = 0.0;
#pragma unroll
        for (int u = 0; u < 2; u++) {   // a row's strips are rarely more than 64
            const int s = u * 32 + lane;
            m2[u] = s < a.strips ? a.pm[row * a.strips + s] : -INFINITY;
            s2[u] = s < a.strips ? a.ps[row * a.strips + s] : 0.0;
            m = fmaxf(m, m2[u]);
        }
        for (int s = 64 + lane; s < a.strips; s += 32) m = fmaxf(m, a.pm[row * a.strips + s]);
        m = warp_max_f32(m);
#pragma unroll
        for (int u = 0; u < 2; u++)
            if (m2[u] > -INFINITY) sum += s2[u] * exp((double)m2[u] - (double)m);
        for (int s = 64 + lane; s < a.strips; s += 32) {
            const float p = a.pm[row * a.strips + s];
            if (p > -INFINITY) sum += a.ps[row * a.strips + s] * exp((double)p - (double)m);
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            row_m[i] = m;
            row_s[i] = log(sum);
            row_cum[i] = cum;
            row_done[i] = done;
        }
    }
    if (t == 0) {
        count = 0;
        bound = -INFINITY;
    }
    // the k-th candidate of a list; the first list of an ended beam is its end token
    auto made = [&](int l, int k, float x, int token) {
        const int beam = (int)a.by_strips.div(l);
        const float cum = row_cum[beam];
        if (!isfinite(cum)) return no_cand();
        if (row_done[beam])
            return k || l != beam * a.strips ? no_cand() : Cand{cum, 0.0f, beam, a.end_token};
        if (token < 0) return no_cand();
        return Cand{(double)cum + (((double)x - row_m[beam]) - row_s[beam]), x, beam, token};
    };
    auto cand = [&](int j) {
        const int l = (int)a.by_n.div(j);
        return made(l, j - l * a.n, a.cx[at + j], a.ct[at + j]);
    };
    auto other = [](const Cand &c, int o) {
        Cand d;
        d.score = __shfl_xor_sync(0xffffffffu, c.score, o);
        d.x = __shfl_xor_sync(0xffffffffu, c.x, o);
        d.beam = __shfl_xor_sync(0xffffffffu, c.beam, o);
        d.token = __shfl_xor_sync(0xffffffffu, c.token, o);
        return d;
    };
    __syncthreads();
    // neighbouring lists, and neighbours of a list, fall into different groups: one beam
    // may be the only good one
    const int groups = a.n <= 8 ? 32 : a.n <= 16 ? 64 : a.n <= 32 ? 128 : 256;
    double best = -INFINITY;
    if (lists >= groups) {
        if (t < lists) best = made(t, 0, head_x, head_t).score;
        for (int l = t + ST; l < lists; l += ST) best = fmax(best, cand(l * a.n).score);
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = t + u * ST, l = (int)a.by_n.div(j);
            if (j < lists * a.n) best = fmax(best, made(l, j - l * a.n, early_x[u], early_t[u]).score);
        }
        for (int j = t + U * ST; j < lists * a.n; j += ST) best = fmax(best, cand(j).score);
    }
    heads[t] = best;
    __syncthreads();
    if (t < groups) {
        for (int j = t + groups; j < ST; j += groups) best = fmax(best, heads[j]);
        tops[t] = best;
    }
    __syncthreads();
    if (t < groups && best > -INFINITY) {
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < groups; j++) rank += tops[j] > best || (tops[j] == best && j < t);
        if (rank == a.n - 1) bound = best;
    }
    __syncthreads();
    double low = bound;
    auto enter = [&](const Cand &c) {
        if (c.beam != INT_MAX && c.score >= low) {
            const int i = atomicAdd(&count, 1);
            if (i < LIST) {
                list[i] = c;
                list_score[i] = c.score;
            }
        }
    };
    int got;
    for (;;) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = t + u * ST, l = (int)a.by_n.div(j);
            if (j < lists * a.n) enter(made(l, j - l * a.n, early_x[u], early_t[u]));
        }
#pragma unroll 4
        for (int j = t + U * ST; j < lists * a.n; j += ST) enter(cand(j));
        __syncthreads();
        got = count;
        if (got <= LIST) break;
        // One beam is far ahead: the n-th best of those that found a place is a nearer
        // bound, unless it is tied.
        for (int i = t; i < LIST; i += ST) {
            const double mine = list_score[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < LIST; j++) rank += list_score[j] > mine || (list_score[j] == mine && j < i);
            if (rank == a.n - 1) bound = mine;
        }
        __syncthreads();
        if (bound == low) break;
        low = bound;
        if (t == 0) count = 0;
        __syncthreads();
    }
    const long long o = (long long)b * a.n;
    auto put = [&](int k, const Cand &c) {
        a.score_out[o + k] = c.beam == INT_MAX ? -INFINITY : (float)c.score;
        a.parent_out[o + k] = c.beam == INT_MAX ? -1 : c.beam;
        a.token_out[o + k] = c.beam == INT_MAX ? -1 : c.token;
    };
    if (got <= LIST) {
        int lanes = 1;   // that share the counting for one candidate
        while (lanes < 32 && got * lanes * 2 <= ST) lanes <<= 1;
        const int part = t & (lanes - 1);
        for (int i0 = 0; i0 < got; i0 += ST / lanes) {
            const int i = i0 + t / lanes;
            const double mine = i < got ? list_score[i] : INFINITY;
            int rank = 0, same = 0;
#pragma unroll 8
            for (int j = part; j < got; j += lanes) {
                rank += list_score[j] > mine;
                same += list_score[j] == mine;
            }
            for (int o = 1; o < lanes; o <<= 1) {
                rank += __shfl_xor_sync(0xffffffffu, rank, o);
                same += __shfl_xor_sync(0xffffffffu, same, o);
            }
            if (part || i >= got || rank >= a.n) continue;
            const Cand c = list[i];
            if (same > 1)   // ties, rarely: by the rest of their order
                for (int j = 0; j < got; j++) rank += list_score[j] == mine && before(list[j], c);
            if (rank < a.n) put(rank, c);
        }
        for (int k = got + t; k < a.n; k += ST) put(k, no_cand());
        return;
    }
    Cand last{INFINITY, INFINITY, -1, -1};   // too many ties for the list: one by one
    for (int k = 0; k < a.n; k++) {
        Cand mine = no_cand();
        for (int j = t; j < lists * a.n; j += ST) {
            const Cand c = cand(j);
            if (before(last, c) && before(c, mine)) mine = c;
        }
        for (int off = 16; off > 0; off >>= 1) {
            const Cand c = other(mine, off);
            if (before(c, mine)) mine = c;
        }
        __syncthreads();
        if (lane == 0) list[warp] = mine;
        __syncthreads();
        last = list[0];
        for (int w = 1; w < ST / 32; w++)
            if (before(list[w], last)) last = list[w];
        if (t == 0) put(k, last);
    }
}

// Logits of a strip.  Where long ones would keep fewer than half the SMs busy: short
// ones (over 129280 tokens of f32 one beam 6.6 us, long 8.0; 1 x 4 beams 7.3 and 8.5,
// bf16 7.4 and 8.9).  Otherwise long ones, whose candidates are fewer to join (1 x 8
// beams 8.9 us, short 9.6; 32 x 8 56 and 74).
int strip_of(size_t rows, size_t vocab) {
    return rows * ((vocab + ST * 32 - 1) / (ST * 32)) < (size_t)num_sms() / 2 ? ST * 16 : ST * 32;
}
size_t strip_count(size_t vocab, int strip) { return (vocab + strip - 1) / strip; }

struct SelectSizes {
    size_t cx, ct, pm, ps, total;
};
SelectSizes select_sizes(size_t rows, size_t vocab, size_t n) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    const size_t parts = rows * strip_count(vocab, strip_of(rows, vocab));
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
    int beams, width;
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
// Loads are issued in groups ahead of their stores: the copies are short, so
// their latency is what they cost.  256 rows, 4 layers of 8 heads of 128 in bf16, pages
// of 64, with weights, 332 MB: 60 us (5.5 TB/s); 4 rows, 12 layers: 3.1 us.
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderArgs a) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.y, lh = blockIdx.x, t = threadIdx.x;
    const int layer = lh / a.c.kv_heads, h = lh - layer * a.c.kv_heads;
    const int src = reorder_source(a, i), n = reorder_len(a, src);
    const int full = a.c.page_div.div(n), rest = n - full * a.c.page_size;
    const int32_t *pages = a.c.table + (int64_t)(src < 0 ? 0 : src) * a.c.table_stride;
    const int here = a.fresh[i];
    const int from = rest > 0 ? pages[full] : -1;
    // a tail whose page is not in the pool stays without one, so that its row goes on
    // giving NaN and not what the fresh page holds
    const bool lost = rest > 0 && (uint32_t)from >= (uint32_t)a.c.n_pages;
    if (lh == 0) {
        for (int j = t; j < a.c.max_pages; j += 256)
            a.table_out[(int64_t)i * a.c.max_pages + j] = j < full ? pages[j] : j == full && !lost ? here : -1;
        if (t == 0) a.lens_out[i] = n;
    }
    if ((uint32_t)from < (uint32_t)a.c.n_pages && (uint32_t)here < (uint32_t)a.c.n_pages) {
        const int64_t at = layer * a.layer_stride + h * a.c.head_stride;
        const int64_t s = at + from * a.c.page_stride, d = at + here * a.c.page_stride;
        const int chunks = rest * (a.c.row_bytes / 16);
        const uint4 *ks = (const uint4 *)(a.c.k + s), *vs = (const uint4 *)(a.c.v + s);
        uint4 *kd = (uint4 *)(a.c.k + d), *vd = (uint4 *)(a.c.v + d);
        for (int x0 = t; x0 < chunks; x0 += 1024) {
            uint4 k[4], v[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (x0 + u * 256 < chunks) {
                    k[u] = ks[x0 + u * 256];
                    v[u] = vs[x0 + u * 256];
                }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (x0 + u * 256 < chunks) {
                    kd[x0 + u * 256] = k[u];
                    vd[x0 + u * 256] = v[u];
                }
        }
    }
    if (a.w) {
        const float *w = a.w + layer * a.w_layer + (src < 0 ? 0 : src) * a.w_row + h * a.w_head;
        const int live = min(n, a.width);
        float *o = a.w_out + layer * a.wo_layer + ((int64_t)i * a.c.kv_heads + h) * a.width;
        for (int x0 = t; x0 < a.width; x0 += 2048) {
            float y[8];
#pragma unroll
            for (int u = 0; u < 8; u++) y[u] = x0 + u * 256 < live ? w[x0 + u * 256] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (x0 + u * 256 < a.width) o[x0 + u * 256] = y[u];
        }
    }
}

}  // namespace
}  // namespace focr

using namespace focr;

extern "C" {

int focr_beam_select_workspace(size_t batch, size_t beams, size_t vocab, size_t n, size_t *bytes) {
    return guarded("beam_select_workspace", [&]() -> int {
        if (!bytes) return fail(FOCR_E_ARG, "beam_select_workspace: null pointer");
        if (beams > MAX_N || n > MAX_N)
            return fail(FOCR_E_UNSUPPORTED, "beam_select_workspace: beams and n are at most " + std::to_string(MAX_N) +
                                                ", not " + std::to_string(beams) + " and " + std::to_string(n));
        size_t rows, x;
        if (!checked_mul(batch, beams, &rows) || !checked_mul(rows, vocab / ST + 8, &x) || x > SIZE_MAX / 1024)
            return fail(FOCR_E_SHAPE, "beam_select_workspace: size out of range");
        *bytes = select_sizes(rows, vocab, n).total;
        return FOCR_OK;
    });
}

int focr_beam_select(const focr_beam_select_args *args, void *stream) {
    return guarded("beam_select", [&]() -> int {
        if (!args) return fail(FOCR_E_ARG, "beam_select: null arguments");
        const void *logits = args->logits;
        const float *scores = args->scores;
        const uint8_t *done = args->done;
        float *scores_out = args->scores_out;
        int32_t *parent_out = args->parent_out;
        int32_t *token_out = args->token_out;
        void *workspace = args->workspace;
        const size_t batch = args->batch;
        const size_t beams = args->beams;
        const size_t vocab = args->vocab;
        const size_t row_stride = args->row_stride;
        const size_t n = args->n;
        const size_t workspace_bytes = args->workspace_bytes;
        const int dtype = args->dtype;
        const int32_t end_token = args->end_token;
        if (dtype != FOCR_F32 && dtype != FOCR_F16 && dtype != FOCR_BF16)
            return fail(FOCR_E_ARG, "beam_select: unknown logits type " + std::to_string(dtype));
        if (beams == 0 || vocab == 0 || n == 0)
            return fail(FOCR_E_SHAPE, "beam_select: beams, vocab and n must not be 0");
        if (beams > MAX_N || n > MAX_N)
            return fail(FOCR_E_UNSUPPORTED, "beam_select: beams and n are at most " + std::to_string(MAX_N));
        if (vocab > (size_t)INT32_MAX - (1 << 20) || batch > (size_t)65535 / beams)
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
        const int strip = strip_of(batch * beams, vocab);
        a.strips = (int)strip_count(vocab, strip);
        a.end_token = end_token;
        a.by_n = FastDiv((uint32_t)n);
        a.by_strips = FastDiv((uint32_t)a.strips);
        char *ws = (char *)workspace;
        a.ps = (double *)ws;
        a.cx = (float *)(ws + sz.ps);
        a.ct = (int32_t *)(ws + sz.ps + sz.cx);
        a.pm = (float *)(ws + sz.ps + sz.cx + sz.ct);
        cudaStream_t st = (cudaStream_t)stream;
        const dim3 grid(a.strips, (unsigned)(batch * beams));
        const bool few = strip == ST * 16;
        auto *part = dtype == FOCR_F32 ? (few ? select_part_kernel<float, 16> : select_part_kernel<float, 32>)
                   : dtype == FOCR_F16 ? (few ? select_part_kernel<__half, 16> : select_part_kernel<__half, 32>)
                                       : (few ? select_part_kernel<__nv_bfloat16, 16> : select_part_kernel<__nv_bfloat16, 32>);
        FOCR_CUDA_TRY(launch_pdl(part, grid, ST, 0, st, a));
        FOCR_CUDA_TRY(launch_pdl(select_join_kernel, (unsigned)batch, ST, 0, st, a));
        return FOCR_OK;
    });
}

int focr_beam_reorder(const focr_paged_cache *cache, const focr_beam_reorder_args *args, void *stream) {
    return guarded("beam_reorder", [&]() -> int {
        if (!args) return fail(FOCR_E_ARG, "beam_reorder: null arguments");
        const int32_t *lens = args->lens;
        const int32_t *parent = args->parent;
        const int32_t *fresh = args->fresh;
        int32_t *table_out = args->table_out;
        int32_t *lens_out = args->lens_out;
        const float *weights = args->weights;
        float *weights_out = args->weights_out;
        const size_t layers = args->layers;
        const size_t layer_stride = args->layer_stride;
        const size_t batch = args->batch;
        const size_t beams = args->beams;
        const size_t width = args->width;
        const size_t weights_layer_stride = args->weights_layer_stride;
        const size_t weights_row_stride = args->weights_row_stride;
        const size_t weights_head_stride = args->weights_head_stride;
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
        if (rows > 65535 || !checked_mul(layers, cache->kv_heads, &lh) || lh > INT32_MAX || width > (1u << 30))
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
        a.beams = (int)beams;
        a.width = (int)width;
        FOCR_CUDA_TRY(launch_pdl(beam_reorder_kernel, dim3((unsigned)lh, (unsigned)rows), 256, 0,
                                 (cudaStream_t)stream, a));
        return FOCR_OK;
    });
}

}  // extern "C"
