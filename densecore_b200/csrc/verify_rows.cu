// Verification of the drafted tokens of many requests, and each one's next token, from given uniform numbers (no counterpart in DenseCore; the rule is dc_b200_verify_accept's).
//
//   p_i = softmax(x_i / T) (or given), draft i is accepted if u_i q_i(t_i) < p_i(t_i) and all before it are; with n accepted, the next token is the first, by index, up to which the
//   sum of r = max(0, p_n - q_n) (of p_n behind the last draft, or where r is nothing) is above u_last times the whole
//
// k_verify_stats (logits alone): the rows' maxima and sums of weights, a row cut into parts where there are few; one pass.  k_verify_next: every CTA of a request decides
// n from those for itself, then sums r over its part of row n in tiles of 2048 tokens; the last CTA of the request finds the tile that the draw falls into, and
// in it the token.  So a row that is accepted is read once, and the one drawn from twice (the second time largely from L2).
//
// A token of a large vocabulary has a millionth of the whole or less, so what decides is of 64 bits.  The statistics' weights are not: 2^((x - max) log2(e) / T) in f32, of which one of 2^-m is off by
// 2^-22 and, as scale and exponent are rounded once each, by m 2^-23 (32 bf16 or 16 f32 ones at a time are added in 32 bits, then in 64).  Weighted by themselves the m of up to 2^19 tokens are 15 at the
// most, so that a sum is off by less than 2^-18.  Sums decide on drafts that are further than 2^-16 from their border alone; for another one (one in some 10^4) every CTA of the request
// sums its row again, in 64 bits.
// The row drawn from has 64-bit weights w, for which its sum S is not known before all of them are: with s, the statistics' S, the one pass sums w, the r' = w - s q that are above 0, and the q
// of those, so that S and then sum max(0, w - S q) = sum r' - (S - s) sum q are known behind it.  That holds where r and r' are of one sign: a warp's tokens that have an r' within 2^-16 s q
// of 0 (some eight of 600 groups), or all where S is further than 2^-17 from s, are summed again with S itself.  Weights of f32 and sums of eight in 32 bits took 56.5 us for the 128 requests below, and drew
// one token in 1500 beside the one that 64 bits give; these take 81.
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
// CTAs an SM that rows are cut for.  128 requests of up to 4 drafts, bf16, 151936 tokens: statistics for 8 / 16 / 24 / 32 CTAs 60.5 / 58.7 / 64.5 / 65.3 us (with f32 weights in drawing); drawing for three CTAs, held
// to 80 registers, so that three fit an SM, 81, for four at 64 registers 88.
constexpr int VR_STATS_CTAS = 16, VR_NEXT_CTAS = 3;
constexpr int VR_PROBS = -1;

struct alignas(16) Stat {      // of a part of a row
    double sum;      // of weights against the part's maximum
    float most;
    int first;       // index of the first largest
};

struct Tile {        // of a row drawn from
    double w, r;     // sums of weights, of what is left above the draft
    float q;         // of the draft's probabilities where something is
    int again;       // warps whose share is not in r and q yet, since some of what is left may be of the other sign: a bit each
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
    Tile* sums;                                // [request][tile], where a request has several CTAs
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

// log2(e) / T, rounded: what the statistics' weights of a request go by.  Differences are held to 1e35, at which a weight is 0 for every scale from 1e-30 on: so NaN and -inf have none, and no
// product overflows.
struct Scale {
    float c;
    bool greedy, bent;      // bent: held to another than it is
    double exact;
    __device__ __forceinline__ explicit Scale(float T) {
        greedy = !(T > 0.0f), bent = !(T > 2e-30f && T < 1e30f);
        exact = 1.4426950408889634074 / (double)T;
        c = greedy ? 1.0f : (float)fmin(fmax(exact, 1e-30), 1e30);
    }
    __device__ __forceinline__ float operator()(float x, float most) const { return ex2(fmaxf(x - most, -1e35f) * c); }      // x at or below `most`, which is finite
};
// The statistics' weights with one multiply-add each: 2^(c x - hi) where c most = hi + lo exactly, so that each is 2^lo fold and a sum of them to be taken 2^-lo fold.  For products that leave lo below 1/32;
// NaN stays NaN.
struct Quick {
    float hi, lo;
    bool is;
    __device__ __forceinline__ Quick(const Scale& c, float most) : hi(c.c * most), lo(fmaf(c.c, most, -hi)), is(fabsf(hi) < 1048576.0f) {}
};
// Weights in 64 bits: t = (x - most) log2(e) / T is off by some 2^-52 of itself, so that a weight of 2^-m is by m 2^-52.  2^t as in P. T. P. Tang's table-driven method (1989): t = n / 32 + f, |f| <= 1/64,
// 2^(n / 32) from a table of 32, which lie in a warp's lanes, 2^f by its Taylor polynomial of degree 5 (what is left out is below 2^-48).  NaN and -inf have no weight, nor has what is below
// 2^-1021; beside an infinite largest only infinite ones have.
struct Exact {
    double c, most, mine;      // mine: 2^(lane / 32)
    bool inf;
    __device__ __forceinline__ Exact(double c_, float m) : c(c_), most(m), mine(exp2((threadIdx.x & 31) / 32.0)), inf(m == INFINITY) {}
    // (by whole warps; beside a finite largest)
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double MAGIC = 0x1.8p47, L = 0.69314718055994530942;
        const double t = ((double)x - most) * c, z = t + MAGIC, f = t - (z - MAGIC);
        const int n = __double2loint(z);
        double y = fma(f, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
        y = fma(f, y, L * L * L / 6.0);
        y = fma(f, y, L * L / 2.0);
        y = fma(f, y, L);
        y = fma(f, y, 1.0) * __shfl_sync(0xffffffffu, mine, n & 31);
        return t > -1021.0 ? __hiloint2double(__double2hiint(y) + (n >> 5) * (1 << 20), __double2loint(y)) : 0.0;
    }
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

// A double of every warp's lane, summed in the order of the warps; to all threads.
__device__ __forceinline__ double cta_sum(double v, double* warps) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < VR_T / 32; ++w) all += warps[w];
    return all;
}

// One CTA per (request, part of the row drawn from).  Bound: issue slots for many requests' logits (some 40 instructions a token, 14 of them of 64 bits, at 60 % of the slots), HBM for probabilities; latency
// for few: the rows' statistics, the decisions, the part, the ticket and the draw's tile one after the other.  One request's whole call, with the statistics: 15 us; 78 MB of
// probabilities: 19.3.  Sums of w and r reduced one after the other: 84 us for the 128 requests.
template <typename TX, bool PROBS>
__global__ void __launch_bounds__(VR_T, 3) k_verify_next(const VerifyParams p) {
    constexpr int WARPS = VR_T / 32;
    __shared__ Stat rows[VR_DRAFTS + 1];
    __shared__ int s_good[VR_DRAFTS], s_n, s_tile, s_last, s_token, s_at_most;
    __shared__ Tile s_sums[VR_TILES];
    __shared__ double s_w[VR_TILES][WARPS], s_r[VR_TILES][WARPS], s_total, s_before, s_warps[WARPS];
    __shared__ float s_q[VR_TILES][WARPS];      // below 0: some of what is left may be of the other sign
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
    const Scale c(PROBS || !p.temperature ? 1.0f : p.temperature[r]);
    if constexpr (!PROBS) {
        for (int i = warp; i <= n; i += WARPS) {
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
    double my_w = 0.0, uq = 0.0;      // the draft's weight, or what is given
    if (tid < n) {
        int good = 0;      // 2: too close to tell by the statistics
        if (inside) {
            if (!(my_q > 0.0f && my_q <= 3.4028235e38f)) my_q = 0.0f;
            uq = (double)my_u * (double)my_q;      // (exact)
            if constexpr (PROBS) {
                good = uq < (my_x > 0.0f && my_x <= 3.4028235e38f ? (double)my_x : 0.0);
            } else {
                const Stat& s = rows[tid];
                if (s.most > -INFINITY) {
                    if (c.greedy) {
                        good = uq < (my_token == s.first ? 1.0 : 0.0);
                    } else {
                        if (s.most == INFINITY) my_w = weight_inf(my_x);
                        else if (my_x > -INFINITY) my_w = exp2(((double)my_x - (double)s.most) * c.exact);
                        good = uq * s.sum < my_w;
                        if (s.most < INFINITY && uq > 0.0 && my_w > 0.0 && (c.bent || fabs(uq * s.sum - my_w) <= 0x1p-16 * my_w)) good = 2;
                    }
                }
            }
        }
        s_good[tid] = good;
    }
    auto first_not_good = [&]() {      // to everyone
        __syncthreads();
        if (tid == 0) {
            int k = 0;
            while (k < n && s_good[k] == 1) ++k;
            s_n = k;
        }
        __syncthreads();
        return s_n;
    };
    int k = first_not_good();
    struct Loaded {
        Eight<TX> x;
        Eight<float> q;
    };
    const int tiles = (p.V + VR_TILE - 1) / VR_TILE;
    if constexpr (!PROBS) {
        while (k < n && s_good[k] == 2) {
            const Exact weight(c.exact, rows[k].most);
            double sum = 0.0;
#pragma unroll 1
            for (int t = 0; t < tiles; ++t) {
                Eight<TX> v;
                float x[8];
                v.load(target + (size_t)k * p.ld, t * VR_TILE + VR_PER * tid, p.V, -INFINITY);
                v.values(x);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += weight(x[i]);
            }
            sum = cta_sum(sum, s_warps);
            if (tid == k) s_good[k] = uq * sum < my_w;
            k = first_not_good();
        }
    }
    // ---- what is drawn from, of eight neighbouring tokens
    const int own = k < n ? p.tokens[(size_t)k * p.R + r] : -1;
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
    const Exact weight(c.exact, st.most);
    auto fetch = [&](int i, bool residual, Loaded& z) {
        z.x.load(row, i, p.V, PROBS ? 0.0f : -INFINITY);
        if (residual && qrow) z.q.load(qrow, i, p.V, 0.0f);
    };
    auto weigh = [&](const Loaded& z, double (&w)[8]) {
        float x[8];
        z.x.values(x);
        if (PROBS || weight.inf) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = !PROBS ? weight_inf(x[j]) : x[j] > 0.0f && x[j] <= 3.4028235e38f ? x[j] : 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = weight(x[j]);
        }
    };
    auto drafted = [&](int i, const Loaded& z, float (&q)[8]) {
        if (qrow) {
            z.q.values(q);
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(q[j]));
            if (top > 0x7F7FFFFFu) {      // below 0, infinite or NaN
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = fmaxf(q[j] <= 3.4028235e38f ? q[j] : 0.0f, 0.0f);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = i + j == own ? 1.0f : 0.0f;
        }
    };
    const int from = part * p.part_tiles, to = min(tiles, from + p.part_tiles);
    {      // every warp's share of each tile
        const bool residual = k < n;
        constexpr int B = PROBS ? 2 : 1;      // tiles on their way at once (probabilities 19.3 us for 22.9 of one; 64-bit weights leave no registers for two: 84 for 81)
        Loaded next[B];
        auto begin = [&](int t) {
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (t + b < to) fetch((t + b) * VR_TILE + VR_PER * tid, residual, next[b]);
        };
        auto add_up = [&](int t, const Loaded& z) {
            double w[8], sw = 0.0, sr = 0.0;
            float sq = 0.0f;
            int nearest = -0x7fffffff;
            weigh(z, w);
            if (!PROBS || !residual) {
#pragma unroll
                for (int j = 0; j < 8; ++j) sw += w[j];
            }
            if (residual) {
                float q[8];
                drafted(t * VR_TILE + VR_PER * tid, z, q);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double left = fma(-st.sum, (double)q[j], w[j]);
                    if (__double2hiint(left) >= 0) {
                        sr += left;
                        if (!PROBS) sq += q[j];
                    }
                    // (|left| <= 2^-16 s q is below 2^-15 w, which the upper halves show)
                    if (!PROBS) nearest = max(nearest, __double2hiint(w[j]) - (__double2hiint(left) & 0x7fffffff));
                }
            }
            if (!PROBS && residual) {      // the lower lanes go on with w, the others with r
                const bool up = lane & 16;
                double mine = up ? sr : sw;
                mine += __shfl_xor_sync(0xffffffffu, up ? sw : sr, 16);
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, x);
                sw = mine, sr = __shfl_down_sync(0xffffffffu, mine, 16);
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, x);
            } else {      // (one of them)
                double mine = residual ? sr : sw;
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, x);
                sw = sr = mine;
            }
            const bool again = !PROBS && __any_sync(0xffffffffu, nearest >= 15 << 20);
            if (lane == 0) s_w[t][warp] = sw, s_r[t][warp] = again ? 0.0 : sr, s_q[t][warp] = again ? -1.0f : sq;
        };
        begin(from);
        for (int t = from; t < to; t += B) {
            Loaded z[B];
#pragma unroll
            for (int b = 0; b < B; ++b) z[b] = next[b];
            begin(t + B);      // (meanwhile)
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (t + b < to) add_up(t + b, z[b]);
        }
        __syncthreads();
    }
    for (int t = from + tid; t < to; t += VR_T) {
        Tile z = {0.0, 0.0, 0.0f, 0};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) z.w += s_w[t][w], z.r += s_r[t][w], z.q += fmaxf(s_q[t][w], 0.0f), z.again |= (s_q[t][w] < 0.0f) << w;
        if (p.parts == 1) s_sums[t] = z;
        else p.sums[(size_t)r * tiles + t] = z;
    }
    __syncthreads();
    if (p.parts > 1) {
        if (tid == 0) {      // (releases what the CTA's threads have stored ahead of the barrier, and acquires what the others' have)
            int before;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.tickets + r) : "memory");
            s_last = before == p.parts - 1;
            if (s_last) p.tickets[r] = 0;
        }
        __syncthreads();
        if (!s_last) return;
        for (int i = tid; i < tiles * (int)(sizeof(Tile) / 8); i += VR_T) reinterpret_cast<double*>(s_sums)[i] = __ldcg(reinterpret_cast<const double*>(p.sums + (size_t)r * tiles) + i);
        __syncthreads();
    }
    // ---- the last CTA of the request: the row's sum, and what is left above the draft by it
    double S = 1.0;
    bool residual = k < n;
    auto left_of = [&](int t, double (&w)[8]) {      // the thread's tokens of a tile
        const int i = t * VR_TILE + VR_PER * tid;
        Loaded z;
        fetch(i, residual, z);
        weigh(z, w);
        if (residual) {
            float q[8];
            drafted(i, z, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = fmax(fma(-S, (double)q[j], w[j]), 0.0);
        }
    };
    // shares of the warps that `which` names of every tile, anew
    auto shares = [&](auto which) {
        for (int t0 = 0; t0 < tiles; t0 += 32)
            for (uint32_t todo = __ballot_sync(0xffffffffu, t0 + lane < tiles && (which(t0 + lane) >> warp & 1)); todo; todo &= todo - 1) {
                const int t = t0 + __ffs(todo) - 1;
                double w[8], sum = 0.0;
                left_of(t, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += w[j];
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (lane == 0) s_r[t][warp] = sum;
            }
        __syncthreads();
    };
    if (!PROBS && residual) {
        double s = 0.0;
        for (int t = tid; t < tiles; t += VR_T) s += s_sums[t].w;
        S = cta_sum(s, s_warps);
        const double more = S - st.sum;
        const bool all = fabs(more) > 0x1p-17 * st.sum;
        auto which = [&](int t) { return all ? (1 << WARPS) - 1 : s_sums[t].again; };
        shares(which);
        for (int t = tid; t < tiles; t += VR_T) {
            Tile& z = s_sums[t];
            double sum = all ? 0.0 : z.r - more * (double)z.q;
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                if (which(t) >> w & 1) sum += s_r[t][w];
            z.r = sum;
        }
    }
    // the tile that the draw falls into, the sums ahead of it, the whole; to everyone
    const float u = p.u[(size_t)r * (p.D + 1) + p.D], uc = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    auto find_tile = [&]() {
        __syncthreads();
        if (warp == 0) {
            const int per = (tiles + 31) / 32, a = min(tiles, lane * per), b = min(tiles, a + per);
            auto sum = [&](int t) { return residual ? s_sums[t].r : s_sums[t].w; };
            double own = 0.0;
            int last = -1;
            for (int t = a; t < b; ++t) {
                own += sum(t);
                if (sum(t) > 0.0) last = t;
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
                for (; t < b && !(before + sum(t) > goal); ++t) before += sum(t);
                if (t >= b) {      // (rounding: the last tile with a weight)
                    t = max(last, 0);
                    before = 0.0;
                    for (int x = 0; x < t; ++x) before += sum(x);
                }
                s_tile = t, s_before = before, s_total = total;
            }
        }
        __syncthreads();
    };
    find_tile();
    if (residual && !(s_total > 0.0)) {      // the draft is nowhere below the target: from the target itself
        residual = false;
        if constexpr (PROBS) {      // (weights have not been summed so far)
            shares([](int) { return (1 << WARPS) - 1; });
            for (int t = tid; t < tiles; t += VR_T) {
                double sum = 0.0;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += s_r[t][w];
                s_sums[t].w = sum;
            }
        }
        find_tile();
    }
    if (tid == 0) s_token = 0x7fffffff, s_at_most = -1;
    __syncthreads();
    if (s_total > 0.0) {
        double w[8];
        const int i0 = s_tile * VR_TILE + VR_PER * tid;
        left_of(s_tile, w);
        double own_sum = 0.0, all;
#pragma unroll
        for (int x = 0; x < 8; ++x) own_sum += w[x];
        // (where rounding leaves none of a thread's tokens above the goal, but their sum is, it is its last with a weight)
        double upto = scan(own_sum, s_warps, all);
        const double goal = (double)uc * s_total - s_before;
        const bool mine = upto + own_sum > goal;
        int found = 0x7fffffff, last = -1;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            upto += w[x];
            if (w[x] > 0.0) last = i0 + x;
            if (upto > goal && w[x] > 0.0) found = min(found, i0 + x);
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
    if ((uintptr_t)target_dev % (type == DC_TYPE_BF16 ? 2 : 4) || ((uintptr_t)draft_probs_dev | (uintptr_t)starts_dev | (uintptr_t)n_drafts_dev | (uintptr_t)draft_tokens_dev | (uintptr_t)temperature_dev |
                                                                       (uintptr_t)uniforms_dev | (uintptr_t)tokens_dev | (uintptr_t)accepted_dev | (uintptr_t)rejected_dev) % 4)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: a buffer is not aligned to its elements");
    // a request's CTAs read these while one of them may have stored its results already
    const size_t each = (size_t)n_requests * 4, out = each * (max_drafts + 1);
    auto meet = [](const void* a, size_t n, const void* b, size_t m) { return a && b && (uintptr_t)a < (uintptr_t)b + m && (uintptr_t)b < (uintptr_t)a + n; };
    const void* const read[] = {starts_dev, n_drafts_dev, temperature_dev};
    for (const void* x : read)
        if (meet(tokens_dev, out, x, each) || meet(accepted_dev, each, x, each) || meet(rejected_dev, each, x, each))
            return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: a result overlaps an input");
    if (meet(rejected_dev, each, tokens_dev, out) || meet(rejected_dev, each, accepted_dev, each)) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "verify_rows: results overlap");
    cudaSetDevice(ctx->device);
    // rows are cut into parts where there are fewer than fill the GPU
    const int tiles = (vocab + VR_TILE - 1) / VR_TILE, n_rows = n_requests * (max_drafts + 1), stat_ctas = VR_STATS_CTAS * ctx->num_sms, next_ctas = VR_NEXT_CTAS * ctx->num_sms;
    int stat_parts = std::min(tiles, (stat_ctas + n_rows - 1) / n_rows), parts = std::min(tiles, (next_ctas + n_requests - 1) / n_requests);
    const int part_tiles = (tiles + parts - 1) / parts, stat_tiles = (tiles + stat_parts - 1) / stat_parts;
    stat_parts = (tiles + stat_tiles - 1) / stat_tiles;
    parts = (tiles + part_tiles - 1) / part_tiles;
    // a workspace of one size, which graphs that hold calls may go on using
    const size_t stats = align256((size_t)(VR_ROWS + stat_ctas) * sizeof(Stat)), sums = align256((size_t)next_ctas * VR_TILES * sizeof(Tile)), tickets = align256((size_t)next_ctas * 4);
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
                            uniforms_dev, tokens_dev, accepted_dev, rejected_dev, (Stat*)ctx->verify_ws, stat_parts, stat_tiles, (Tile*)(ctx->verify_ws + stats), (int32_t*)(ctx->verify_ws + stats + sums)};
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
