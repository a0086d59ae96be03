// Verification of the drafted tokens of many requests, and each one's next token, from given uniform numbers (no counterpart in DenseCore; the rule is dc_b200_verify_accept's).
//
//   p_i = softmax(x_i / T) (or given), draft i is accepted if u_i q_i(t_i) < p_i(t_i) and all before it are; with n accepted, the next token is the first, by index, up to which the
//   sum of r = max(0, p_n - q_n) (of p_n behind the last draft, or where r is nothing) is above u_last times the whole
//
// k_verify_stats (logits alone): the rows' maxima and sums of weights, a row cut into parts where there are few; one pass.  k_verify_next: every CTA of a request decides
// n from those for itself, then sums r over its part of row n in tiles of 2048 tokens; the last CTA of the request finds the tile that the draw falls into, and
// in it the token.  So a row that is accepted is read once, and the one drawn from twice (the second time largely from L2).
// Weights are 2^((x - max) log2(e) / T) in f32: one of 2^-m is off by 2^-22 and, as scale and exponent are rounded once each, by m 2^-23.  Sums are of 64 bits (eight weights at a time in
// 32), in an order that does not depend on timing.
#include <math.h>

#include <algorithm>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_launch.cuh"

using namespace dc;

#define DC_TRY(expr)                       \
    do {                                   \
        int _st = (expr);                  \
        if (_st != DC_B200_OK) return _st; \
    } while (0)

namespace {

constexpr int VR_T = 256, VR_PER = 8, VR_TILE = VR_T * VR_PER, VR_DRAFTS = 64, VR_VOCAB = 389120, VR_TILES = VR_VOCAB / VR_TILE, VR_ROWS = 65536;
// CTAs an SM that rows are cut for.  128 requests of up to 4 drafts, bf16, 151936 tokens: statistics for 8 / 16 / 24 / 32 CTAs 60.5 / 58.7 / 64.5 / 65.3 us, drawing (three fit an SM) for 2 / 3 / 4 58.7 /
// 56.5 / 60.2; 64 requests of 3 drafts, probabilities, drawing 19.5 / 19.9 / 20.8.
constexpr int VR_STATS_CTAS = 16, VR_NEXT_CTAS = 3;
constexpr int VR_PROBS = -1;

struct alignas(16) Stat {      // of a part of a row
    double sum;      // of weights against the part's maximum
    float most;
    int first;       // index of the first largest
};

struct VerifyParams {
    const void* target;
    size_t ld;
    int rows, V, R, D, parts, part_tiles;      // tiles of a part
    const int32_t *starts, *n_drafts, *tokens;
    const float *q, *temperature, *u;
    int32_t *out, *accepted, *rejected;
    Stat* stats;                               // [request][row][stat_parts]
    int stat_parts, stat_tiles;
    double* sums;                              // [request][tile], where a request has several CTAs
    int32_t* tickets;
};

// Drafts of a request and its first row; false: it takes no part.
__device__ __forceinline__ bool request(const VerifyParams& p, int r, int& n, int& row0) {
    n = p.n_drafts ? min(p.n_drafts[r], p.D) : p.D;
    row0 = p.starts ? p.starts[r] : r * (p.D + 1);
    return n >= 0 && row0 >= 0 && (long long)row0 + n < p.rows;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// pairs of f32 in a register pair: two results an instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(a));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }

// log2(e) / T, rounded: what all weights of a request go by.  Differences are held to 1e35, at which a weight is 0 for every scale from 1e-30 on: so NaN and -inf have none, and no
// product overflows.
struct Scale {
    float c;
    bool greedy;
    __device__ __forceinline__ explicit Scale(float T) {
        greedy = !(T > 0.0f);
        c = greedy ? 1.0f : (float)fmin(fmax(1.4426950408889634 / (double)T, 1e-30), 1e30);
    }
    __device__ __forceinline__ float operator()(float x, float most) const { return ex2(fmaxf(x - most, -1e35f) * c); }      // x at or below `most`, which is finite
};
// The same weights with one multiply-add each: 2^(c x - hi) where c most = hi + lo exactly, so that each is 2^lo fold, and 2^-lo undoes it.  For products that leave lo below 1/32; NaN stays NaN.
struct Quick {
    float hi, lo;
    bool is;
    __device__ __forceinline__ Quick(const Scale& c, float most) : hi(c.c * most), lo(fmaf(c.c, most, -hi)), is(fabsf(hi) < 1048576.0f) {}
    __device__ __forceinline__ float operator()(const Scale& c, float x) const { return ex2(fmaf(c.c, x, -hi)); }
};
__device__ __forceinline__ float weight_inf(float x) { return x == INFINITY ? 1.0f : 0.0f; }      // beside an infinite largest

// Eight neighbouring values of a row from index i on, as they lie: one or two loads of sixteen bytes.
template <typename TX>
struct Eight {
    uint4 v[sizeof(TX) / 2];
    __device__ __forceinline__ static bool fits(const TX* row, int i, int V) { return i + 8 <= V && ((uintptr_t)(row + i) & 15) == 0; }
    // `none` behind the row's end
    __device__ __forceinline__ void load(const TX* row, int i, int V, float none) {
        if (fits(row, i, V)) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(TX) / 2; ++k) v[k] = __ldg(reinterpret_cast<const uint4*>(row + i) + k);
        } else {
            alignas(16) TX x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = i + k < V ? row[i + k] : (TX)none;
#pragma unroll
            for (int k = 0; k < (int)sizeof(TX) / 2; ++k) v[k] = reinterpret_cast<const uint4*>(x)[k];
        }
    }
    __device__ __forceinline__ void values(float (&x)[8]) const {
#pragma unroll
        for (int k = 0; k < (int)sizeof(TX) / 2; ++k) {
            const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(TX) == 2) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
                else x[4 * k + j] = __uint_as_float(w[j]);
            }
        }
    }
};

// Two parts of a row as one: sums against the larger maximum, the first largest.
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, const Scale& c) {
    Stat s;
    s.most = fmaxf(a.most, b.most);
    s.first = a.most == b.most ? min(a.first, b.first) : a.most > b.most ? a.first : b.first;
    // (the weight of a maximum against itself is 1, also of an infinite one; beside that others have none)
    const float f = a.most == b.most ? 1.0f : s.most == INFINITY ? 0.0f : c(fminf(a.most, b.most), s.most);
    s.sum = a.most == s.most ? a.sum + b.sum * (double)f : a.sum * (double)f + b.sum;
    return s;
}
// Those of a warp's lanes, to all of them.
__device__ __forceinline__ Stat warp_join(const Stat& a, const Scale& c) {
    Stat s;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(s.most) : "f"(a.most));
    s.first = c.greedy ? __reduce_min_sync(0xffffffffu, a.most == s.most ? a.first : 0x7fffffff) : 0x7fffffff;
    s.sum = a.most == s.most ? a.sum : s.most == INFINITY ? 0.0 : a.sum * (double)c(a.most, s.most);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, k);      // (the same in all lanes: sums of two are commutative)
    return s;
}

// One CTA per (row, part).  Bound: issue slots (64 %, exponentials 53 % of their pipe's) ahead of HBM: 141 MB of bf16 rows in 40 us, 3.5 TB/s (a call of 63 us; without
// divisions and with maxima joined at once 59).  Four tiles on their way at 64 registers (four CTAs an SM); two tiles and five or six CTAs 67 to 68 for 66.
template <typename TX>
__global__ void __launch_bounds__(VR_T, 4) k_verify_stats(const VerifyParams p) {
    constexpr int B = sizeof(TX) == 2 ? 4 : 2;      // tiles on their way at once
    __shared__ Stat warps[VR_T / 32];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x, i = blockIdx.y, part = blockIdx.z;
    const float T = p.temperature ? p.temperature[r] : 1.0f;
    int n, row0;
    if (!request(p, r, n, row0) || i > n) return;
    const TX* row = reinterpret_cast<const TX*>(p.target) + (size_t)(row0 + i) * p.ld;
    const int first = part * p.stat_tiles, last = min((p.V + VR_TILE - 1) / VR_TILE, first + p.stat_tiles);
    float most = -INFINITY;
    int where = 0x7fffffff;      // of a request that goes by the largest alone
    double sum = 0.0;
    Eight<TX> next[B];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int b = 0; b < B; ++b) next[b].load(row, t0 + b < last ? (t0 + b) * VR_TILE + VR_PER * (int)threadIdx.x : p.V, p.V, -INFINITY);
    };
    if (first < last) fetch(first);
    const Scale c(T);
    for (int t0 = first; t0 < last; t0 += B) {
        float x[B][8], top = -INFINITY;
        if constexpr (sizeof(TX) == 2) {      // (pairs as they lie)
            __nv_bfloat162 m = __floats2bfloat162_rn(-INFINITY, -INFINITY);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const uint32_t w[4] = {next[b].v[0].x, next[b].v[0].y, next[b].v[0].z, next[b].v[0].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(w + k));
            }
            top = fmaxf(__low2float(m), __high2float(m));
        }
#pragma unroll
        for (int b = 0; b < B; ++b) next[b].values(x[b]);
        if (t0 + B < last) fetch(t0 + B);      // (on their way meanwhile)
        if constexpr (sizeof(TX) == 4) {
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int k = 0; k < 8; ++k) top = fmaxf(top, x[b][k]);
        }
        if (top > most) {
            sum = most > -INFINITY && top < INFINITY ? sum * (double)c(most, top) : 0.0;
            most = top;
            if (c.greedy) {
#pragma unroll
                for (int b = B - 1; b >= 0; --b)
#pragma unroll
                    for (int k = 7; k >= 0; --k)
                        if (x[b][k] == top) where = (t0 + b) * VR_TILE + VR_PER * (int)threadIdx.x + k;
            }
        }
        if (!(top > -INFINITY) || c.greedy) continue;      // nothing with a weight, or nobody asks for it
        float all = 0.0f;
        const Quick q(c, most);
        if (q.is) {
            uint64_t s[2] = {0, 0};      // (two sums of pairs)
            const uint64_t c2 = pair(c.c, c.c), h2 = pair(-q.hi, -q.hi);
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const float2 y = unpair(fma2(pair(x[b][k], x[b][k + 1]), c2, h2));
                    s[k / 2 & 1] = add2(s[k / 2 & 1], pair(ex2(y.x), ex2(y.y)));
                }
            const float2 z = unpair(add2(s[0], s[1]));
            all = (z.x + z.y) * ex2(-q.lo);
        }
        if (!(q.is && all < INFINITY)) {      // an infinite largest, a product too large, or a NaN among them
            all = 0.0f;
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int k = 0; k < 8; ++k) all += most == INFINITY ? weight_inf(x[b][k]) : c(x[b][k], most);
        }
        sum += (double)all;
    }
    Stat s;
    s.sum = sum, s.most = most, s.first = where;
    s = warp_join(s, c);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s.sum = 0.0, s.most = -INFINITY, s.first = 0x7fffffff;
        if (threadIdx.x < VR_T / 32) s = warps[threadIdx.x];
        s = warp_join(s, c);
        if (threadIdx.x == 0) p.stats[((size_t)r * (p.D + 1) + i) * p.stat_parts + part] = s;
    }
}

// Exclusive sum over the CTA's threads.
__device__ __forceinline__ double scan(double v, double* warps, double& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double in = v;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, in, s);
        if (lane >= s) in += o;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = in;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
#pragma unroll
    for (int w = 0; w < VR_T / 32; ++w) {
        if (w == warp) before = all;
        all += warps[w];
    }
    const double ex = __shfl_up_sync(0xffffffffu, in, 1);
    return before + (lane ? ex : 0.0);
}

// One CTA per (request, part of the row drawn from).  Bound: HBM for many requests (the row and its draft's probabilities, once; the draw's own tile again), latency for few: the rows'
// statistics, the decisions, the part, the ticket and the draw's tile one after the other.  78 MB of probabilities: 19.5 us (4.0 TB/s); held to 64 registers, so that four CTAs fit an SM,
// it spills: 23 to 29.  One request's whole call, with the statistics: 11.6 us.
template <typename TX, bool PROBS>
__global__ void __launch_bounds__(VR_T) k_verify_next(const VerifyParams p) {
    __shared__ Stat rows[VR_DRAFTS + 1];
    __shared__ int s_good[VR_DRAFTS], s_n, s_tile, s_last, s_token, s_at_most;
    __shared__ double s_sums[VR_TILES], s_warps[VR_TILES][VR_T / 32], s_total, s_before;
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x / p.parts, part = blockIdx.x % p.parts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int n, row0;
    if (!request(p, r, n, row0)) {
        if (part == 0) {
            for (int i = tid; i <= p.D; i += VR_T) p.out[(size_t)r * (p.D + 1) + i] = -1;
            if (tid == 0) {
                p.accepted[r] = 0;
                if (p.rejected) p.rejected[r] = 0;
            }
        }
        return;
    }
    const TX* target = reinterpret_cast<const TX*>(p.target) + (size_t)row0 * p.ld;
    // ---- the drafts, a thread each: what decides on them, but for the rows' statistics, is on its way meanwhile
    static_assert(VR_DRAFTS <= VR_T, "a thread a draft");
    const int my_token = tid < n ? p.tokens[(size_t)tid * p.R + r] : -1;
    const bool inside = my_token >= 0 && my_token < p.V;
    float my_q = inside && p.q ? p.q[((size_t)tid * p.R + r) * p.V + my_token] : 1.0f;
    const float my_x = inside ? value(target[(size_t)tid * p.ld + my_token]) : 0.0f, my_u = tid < n ? p.u[(size_t)r * (p.D + 1) + tid] : 0.0f;
    const Scale c(PROBS ? 1.0f : p.temperature ? p.temperature[r] : 1.0f);
    if constexpr (!PROBS) {
        for (int i = warp; i <= n; i += VR_T / 32) {
            Stat s;
            s.sum = 0.0, s.most = -INFINITY, s.first = 0x7fffffff;
            const Stat* from = p.stats + ((size_t)r * (p.D + 1) + i) * p.stat_parts;
            for (int k = lane; k < p.stat_parts; k += 32) {
                Stat o;
                const int4 v = __ldcg(reinterpret_cast<const int4*>(from + k));
                o.sum = __hiloint2double(v.y, v.x), o.most = __int_as_float(v.z), o.first = v.w;
                s = join(s, o, c);
            }
            s = warp_join(s, c);
            if (lane == 0) rows[i] = s;
        }
        __syncthreads();
    }
    if (tid < n) {
        bool good = false;
        if (inside) {
            if (!(my_q > 0.0f && my_q <= 3.4028235e38f)) my_q = 0.0f;
            const double uq = (double)my_u * (double)my_q;
            if constexpr (PROBS) {
                good = uq < (my_x > 0.0f && my_x <= 3.4028235e38f ? (double)my_x : 0.0);
            } else {
                const Stat& s = rows[tid];
                if (s.most > -INFINITY)
                    good = c.greedy ? uq < (my_token == s.first ? 1.0 : 0.0) : uq * s.sum < (double)(s.most == INFINITY ? weight_inf(my_x) : c(my_x, s.most));
            }
        }
        s_good[tid] = good;
    }
    __syncthreads();
    if (tid == 0) {
        int k = 0;
        while (k < n && s_good[k]) ++k;
        s_n = k;
    }
    __syncthreads();
    // ---- what is drawn from, of eight neighbouring tokens
    const int k = s_n, own = k < n ? p.tokens[(size_t)k * p.R + r] : -1;
    const TX* row = target + (size_t)k * p.ld;
    const float* qrow = k < n && p.q ? p.q + ((size_t)k * p.R + r) * p.V : nullptr;
    auto answer = [&](int token) {      // by the whole CTA
        for (int i = tid; i <= p.D; i += VR_T) p.out[(size_t)r * (p.D + 1) + i] = i < k ? p.tokens[(size_t)i * p.R + r] : i == k ? token : -1;
        if (tid == 0) {
            p.accepted[r] = k;
            if (p.rejected) p.rejected[r] = n - k;
        }
    };
    Stat st;
    st.sum = 1.0, st.most = 0.0f, st.first = 0;
    if constexpr (!PROBS) {
        st = rows[k];
        if (c.greedy || !(st.most > -INFINITY)) {      // all on one token, which stays whatever the draft had on it; or nothing
            if (part == 0) answer(st.most > -INFINITY ? st.first : -1);
            return;
        }
    }
    const Quick quick(c, st.most);
    const float inv = (float)(1.0 / st.sum), quick_inv = inv * ex2(-quick.lo);
    struct Loaded {
        Eight<TX> x;
        Eight<float> q;
    };
    auto fetch = [&](int i, bool residual, Loaded& z) {
        z.x.load(row, i, p.V, PROBS ? 0.0f : -INFINITY);
        if (residual && qrow) z.q.load(qrow, i, p.V, 0.0f);
    };
    // (a weight that is NaN is below 0 by fmaxf)
    auto drawn_from = [&](int i, bool residual, const Loaded& z, float (&w)[8]) {
        float f = 1.0f, q[8] = {};
        z.x.values(w);
        if constexpr (PROBS) {
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = w[x] <= 3.4028235e38f ? w[x] : 0.0f;
        } else if (quick.is) {
            f = quick_inv;
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = quick(c, w[x]);
        } else {
            f = inv;
#pragma unroll
            for (int x = 0; x < 8; ++x) w[x] = st.most == INFINITY ? weight_inf(w[x]) : c(w[x], st.most);
        }
        if (residual && qrow) {
            z.q.values(q);
#pragma unroll
            for (int x = 0; x < 8; ++x) q[x] = fmaxf(q[x] <= 3.4028235e38f ? q[x] : 0.0f, 0.0f);
        } else if (residual && own >= i && own < i + 8) {
#pragma unroll
            for (int x = 0; x < 8; ++x) q[x] = i + x == own ? 1.0f : 0.0f;
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) w[x] = fmaxf(fmaf(w[x], f, -q[x]), 0.0f);
    };
    auto sum_of = [](const float (&w)[8]) { return (double)(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]))); };
    const int tiles = (p.V + VR_TILE - 1) / VR_TILE, from = part * p.part_tiles, to = min(tiles, from + p.part_tiles);
    auto sum_tiles = [&](int from, int to, bool residual) {      // every warp's share of each tile
        constexpr int B = 2;
        Loaded next[B];
        auto begin = [&](int t) {
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (t + b < to) fetch((t + b) * VR_TILE + VR_PER * tid, residual, next[b]);
        };
        begin(from);
        for (int t = from; t < to; t += B) {
            double s[B];
            Loaded z[B];
#pragma unroll
            for (int b = 0; b < B; ++b) z[b] = next[b];
            begin(t + B);      // (on their way meanwhile)
#pragma unroll
            for (int b = 0; b < B; ++b) {
                float w[8];
                drawn_from((t + b) * VR_TILE + VR_PER * tid, residual, z[b], w);
                s[b] = sum_of(w);
            }
#pragma unroll
            for (int x = 16; x > 0; x >>= 1)
#pragma unroll
                for (int b = 0; b < B; ++b) s[b] += __shfl_xor_sync(0xffffffffu, s[b], x);
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (lane == 0 && t + b < to) s_warps[t + b][warp] = s[b];
        }
        __syncthreads();
    };
    auto tile_sum = [&](int t) {
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < VR_T / 32; ++w) s += s_warps[t][w];
        return s;
    };
    const float u = p.u[(size_t)r * (p.D + 1) + p.D], uc = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    auto find_tile = [&]() {      // to everyone: the tile that the draw falls into, the sums ahead of it, the whole
        __syncthreads();
        if (warp == 0) {
            const int per = (tiles + 31) / 32, a = min(tiles, lane * per), b = min(tiles, a + per);
            double own = 0.0;
            int last = -1;
            for (int t = a; t < b; ++t) {
                own += s_sums[t];
                if (s_sums[t] > 0.0) last = t;
            }
            double upto = own;
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, upto, x);
                if (lane >= x) upto += o;
            }
            const double total = __shfl_sync(0xffffffffu, upto, 31), goal = (double)uc * total;
            last = __reduce_max_sync(0xffffffffu, last);
            const uint32_t there = __ballot_sync(0xffffffffu, upto > goal);
            if (lane == (there ? __ffs(there) - 1 : 31)) {
                double before = upto - own;
                int t = a;
                for (; t < b && !(before + s_sums[t] > goal); ++t) before += s_sums[t];
                if (t >= b) {      // (rounding: the last tile with a weight)
                    t = max(last, 0);
                    before = 0.0;
                    for (int x = 0; x < t; ++x) before += s_sums[x];
                }
                s_tile = t, s_before = before, s_total = total;
            }
        }
        __syncthreads();
    };
    sum_tiles(from, to, k < n);
    for (int t = from + tid; t < to; t += VR_T) {
        const double s = tile_sum(t);
        if (p.parts == 1) s_sums[t] = s;
        else p.sums[(size_t)r * tiles + t] = s;
    }
    if (p.parts > 1) {
        __syncthreads();
        if (tid == 0) {      // (releases what the CTA's threads have stored ahead of the barrier, and acquires what the others' have)
            int before;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.tickets + r) : "memory");
            s_last = before == p.parts - 1;
            if (s_last) p.tickets[r] = 0;
        }
        __syncthreads();
        if (!s_last) return;
        for (int t = tid; t < tiles; t += VR_T) s_sums[t] = __ldcg(p.sums + (size_t)r * tiles + t);
    }
    bool residual = k < n;
    find_tile();
    if (residual && !(s_total > 0.0)) {      // the draft is nowhere below the target: from the target itself
        residual = false;
        sum_tiles(0, tiles, false);
        for (int t = tid; t < tiles; t += VR_T) s_sums[t] = tile_sum(t);
        find_tile();
    }
    if (tid == 0) s_token = 0x7fffffff, s_at_most = -1;
    __syncthreads();
    if (s_total > 0.0) {
        float w[8];
        const int i0 = s_tile * VR_TILE + VR_PER * tid;
        Loaded z;
        fetch(i0, residual, z);
        drawn_from(i0, residual, z, w);
        // (a thread's sum is of f32 sums, those up to each of its tokens are of 64 bits: where rounding leaves none of them above the goal, it is its last with a weight)
        double all, own_sum = sum_of(w), upto = scan(own_sum, s_warps[0], all);
        const double goal = (double)uc * s_total - s_before;
        const bool mine = upto + own_sum > goal;
        int found = 0x7fffffff, last = -1;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            upto += (double)w[x];
            if (w[x] > 0.0f) last = i0 + x;
            if (upto > goal && w[x] > 0.0f) found = min(found, i0 + x);
        }
        if (!mine) found = 0x7fffffff;
        else if (found == 0x7fffffff && last >= 0) found = last;
        found = __reduce_min_sync(0xffffffffu, found), last = __reduce_max_sync(0xffffffffu, last);
        if (lane == 0) atomicMin(&s_token, found), atomicMax(&s_at_most, last);
    }
    __syncthreads();
    answer(s_token < p.V ? s_token : s_at_most);      // (rounding: the tile's last with a weight)
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

template <typename TX, bool PROBS>
int launch(dc_ctx* ctx, const VerifyParams& p) {
    if constexpr (!PROBS)
        DC_TRY(dc_launch(ctx, "k_verify_stats", k_verify_stats<TX>, dim3(p.R, p.D + 1, p.stat_parts), dim3(VR_T), 0, p));
    return dc_launch(ctx, "k_verify_next", k_verify_next<TX, PROBS>, dim3(p.R * p.parts), dim3(VR_T), 0, p);
}

}  // namespace

extern "C" {

int dc_b200_verify_rows_dev(dc_ctx* ctx, const void* target_dev, int type, int64_t ld, int rows, int vocab, int n_requests, int max_drafts, const int32_t* starts_dev,
                            const int32_t* n_drafts_dev, const int32_t* draft_tokens_dev, const float* draft_probs_dev, const float* temperature_dev, const float* uniforms_dev,
                            int32_t* tokens_dev, int32_t* accepted_dev, int32_t* rejected_dev) {
    if (!ctx) return DC_B200_INVALID_ARGUMENT;
    if (ld == 0) ld = vocab;
    if (rows < 0 || vocab < 1 || ld < vocab || n_requests < 0 || max_drafts < 0)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: bad shape (%d requests of %d drafts, %d rows of %d, stride %lld)", n_requests, max_drafts, rows, vocab, (long long)ld);
    if (type != DC_TYPE_F32 && type != DC_TYPE_BF16 && type != VR_PROBS)
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "verify_rows: rows of type %d (F32 and BF16 logits and f32 probabilities, -1, are supported)", type);
    if (vocab > VR_VOCAB || max_drafts > VR_DRAFTS || (long long)n_requests * (max_drafts + 1) > VR_ROWS)
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "verify_rows: %d requests of %d drafts, %d tokens", n_requests, max_drafts, vocab);
    if (n_requests == 0) return DC_B200_OK;
    if (!target_dev || (max_drafts && !draft_tokens_dev) || !uniforms_dev || !tokens_dev || !accepted_dev) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: null buffer");
    if ((uintptr_t)target_dev % (type == DC_TYPE_BF16 ? 2 : 4) || (uintptr_t)draft_probs_dev % 4) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: a buffer is not aligned to its elements");
    cudaSetDevice(ctx->device);
    // rows are cut into parts where there are fewer than fill the GPU
    const int tiles = (vocab + VR_TILE - 1) / VR_TILE, n_rows = n_requests * (max_drafts + 1), stat_ctas = VR_STATS_CTAS * ctx->num_sms, next_ctas = VR_NEXT_CTAS * ctx->num_sms;
    int stat_parts = std::min(tiles, (stat_ctas + n_rows - 1) / n_rows), parts = std::min(tiles, (next_ctas + n_requests - 1) / n_requests);
    const int part_tiles = (tiles + parts - 1) / parts, stat_tiles = (tiles + stat_parts - 1) / stat_parts;
    stat_parts = (tiles + stat_tiles - 1) / stat_tiles;
    parts = (tiles + part_tiles - 1) / part_tiles;
    // a workspace of one size, which graphs that hold calls may go on using
    const size_t stats = align256((size_t)(VR_ROWS + stat_ctas) * sizeof(Stat)), sums = align256((size_t)next_ctas * VR_TILES * sizeof(double)), tickets = align256((size_t)next_ctas * 4);
    if (!ctx->verify_ws) {
        cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(ctx->stream, &st) != cudaSuccess || st != cudaStreamCaptureStatusNone)
            return dc_fail(ctx, DC_B200_UNSUPPORTED, "verify_rows: a context's first call cannot be captured");
        void* ws = nullptr;
        DC_TRY(dc_check_cuda(ctx, cudaMalloc(&ws, stats + sums + tickets), "verify_rows: workspace"));
        const cudaError_t e = cudaMemsetAsync((uint8_t*)ws + stats + sums, 0, tickets, ctx->stream);
        if (e != cudaSuccess) {
            cudaFree(ws);
            return dc_check_cuda(ctx, e, "verify_rows: workspace");
        }
        ctx->verify_ws = (uint8_t*)ws;
    }
    const VerifyParams p = {target_dev, (size_t)ld, rows, vocab, n_requests, max_drafts, parts, part_tiles, starts_dev, n_drafts_dev, draft_tokens_dev, draft_probs_dev, temperature_dev,
                            uniforms_dev, tokens_dev, accepted_dev, rejected_dev, (Stat*)ctx->verify_ws, stat_parts, stat_tiles, (double*)(ctx->verify_ws + stats), (int32_t*)(ctx->verify_ws + stats + sums)};
    return type == VR_PROBS ? launch<float, true>(ctx, p) : type == DC_TYPE_F32 ? launch<float, false>(ctx, p) : launch<__nv_bfloat16, false>(ctx, p);
}

int dc_b200_verify_rows(dc_ctx* ctx, const float* target_host, int n_requests, int vocab, int max_drafts, const int32_t* n_drafts, const int32_t* draft_tokens, const float* draft_probs,
                        const float* temperature, int probs, const float* uniforms, int32_t* tokens_out, int32_t* accepted_out) {
    if (!ctx) return DC_B200_INVALID_ARGUMENT;
    if (!target_host || n_requests < 1 || vocab < 1 || max_drafts < 0 || (max_drafts && !draft_tokens) || !uniforms || !tokens_out || !accepted_out)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: bad argument");
    if (vocab > VR_VOCAB || max_drafts > VR_DRAFTS || (long long)n_requests * (max_drafts + 1) > VR_ROWS)
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "verify_rows: %d requests of %d drafts, %d tokens", n_requests, max_drafts, vocab);
    const size_t rows = (size_t)n_requests * (max_drafts + 1);
    for (size_t i = 0; i < rows; ++i)
        if (!(uniforms[i] >= 0.0f && uniforms[i] < 1.0f)) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: uniform number %zu is out of range", i);
    for (int r = 0; r < n_requests; ++r)
        if ((temperature && !(temperature[r] >= 0.0f)) || (n_drafts && (n_drafts[r] < 0 || n_drafts[r] > max_drafts)))
            return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: request %d has a setting out of range", r);
    cudaSetDevice(ctx->device);
    const size_t target = rows * vocab * 4, drafts = (size_t)n_requests * max_drafts, q = draft_probs ? drafts * vocab * 4 : 0;
    uint8_t* at = dc_scratch(ctx, align256(target) + align256(q) + 6 * align256(rows * 4));
    if (!at) return DC_B200_OUT_OF_MEMORY;
    int st = DC_B200_OK;
    auto up = [&](const void* from, size_t n) -> uint8_t* {      // (pageable sources: the copy is done with them when it returns)
        uint8_t* to = at;
        at += align256(n);
        if (from && n && st == DC_B200_OK) st = dc_check_cuda(ctx, cudaMemcpyAsync(to, from, n, cudaMemcpyHostToDevice, ctx->stream), "verify_rows");
        return from ? to : nullptr;
    };
    const uint8_t *x = up(target_host, target), *pq = up(draft_probs, q), *t = up(draft_tokens, drafts * 4), *nd = up(n_drafts, (size_t)n_requests * 4),
                  *temp = up(temperature, (size_t)n_requests * 4), *u = up(uniforms, rows * 4);
    DC_TRY(st);
    int32_t *tokens = (int32_t*)at, *accepted = (int32_t*)(at + align256(rows * 4));
    DC_TRY(dc_b200_verify_rows_dev(ctx, x, probs ? VR_PROBS : DC_TYPE_F32, 0, (int)rows, vocab, n_requests, max_drafts, nullptr, (const int32_t*)nd, (const int32_t*)t, (const float*)pq,
                                   (const float*)temp, (const float*)u, tokens, accepted, nullptr));
    DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(tokens_out, tokens, rows * 4, cudaMemcpyDeviceToHost, ctx->stream), "verify_rows"));
    DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(accepted_out, accepted, (size_t)n_requests * 4, cudaMemcpyDeviceToHost, ctx->stream), "verify_rows"));
    return dc_b200_synchronize(ctx);
}

}  // extern "C"
