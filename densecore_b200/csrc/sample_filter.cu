// Sampling of one token a row by temperature, top-k, top-p and min-p from given uniform numbers (the order of DenseCore's sampler: temperature, top-k, top-p,
// core/src/sampler/sampler.cpp:235-262; min-p after them).
//
// The order of a row's tokens is by falling logit, equal ones by rising index; every filter keeps a beginning of it, so that one comparison with the last kept
// token's key (value, index) decides.  Weights exp((x - largest) / T) are whole numbers of 2^-44 (made in 64 bits): their sums do not depend on the order of
// additions, so that atomics in any order give the same result, and a border between two tokens moves by 2^-44 times the number of tokens at most.
//
// One cluster of CTAs per row: the row lies in their shared memory, a contiguous part each, and is read from HBM once.
//   a cut by number: the threads' largest tokens, in a histogram of 2048 bins of falling value, give a bin that the cut cannot lie beyond;
//   a cut by weight: a histogram of numbers (32-bit atomics; sums of 64 bits in shared memory took ten times as long) bounds the weights ahead of every bin from both
//   sides, between which the cut lies;
//   up to 1024 tokens down to there: they are sorted in one CTA, which applies all filters and draws;
//   up to here all is bound by latency: one row of 151936 tokens 10.9 us, sixteen with settings of their own 27 to 44 us, by the settings;
//   else the bins between the bounds are refined until 1024 tokens or one value is left, and the part of the row with the draw is searched.
// Bound for many rows by nucleus: issue slots (58 %) and waits for one another between passes over shared memory (weights twice, numbers once, the search): 256 bf16 rows
// 229 us, with their distributions 287 us, 810 GB/s.  By top-k 50 and top-p 0.95 90 and 139 us, by temperature alone 107 and 166.  Two CTAs of 512 threads an SM leave 64
// registers a thread, of which 40 to 64 bytes spill.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_launch.cuh"

namespace cg = cooperative_groups;
using namespace dc;

#define DC_TRY(expr)                       \
    do {                                   \
        int _st = (expr);                  \
        if (_st != DC_B200_OK) return _st; \
    } while (0)

namespace {

typedef unsigned long long u64;
constexpr int SF_T = 512, SF_W = SF_T / 32, SF_BINS = 2048, SF_LIST = 1024, SF_SHORT = 256, SF_NEAR = 64, SF_CLUSTER = 16;
constexpr int SF_GROUPS = 256;          // of a row's threads, 2 n_cta neighbours each
constexpr int SF_MOST = 48 * 1024;      // f32 tokens of a CTA
constexpr int SF_VOCAB = 8 * (SF_MOST - 32 * SF_W);
constexpr u64 SF_ONE = 1ull << 44;

struct SampleParams {
    const void* logits;
    size_t ld;
    int V, seg;      // seg: tokens of a warp, contiguous
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p, *u;
    int32_t* token;
    float *p, *dist;
};

__device__ __forceinline__ uint32_t sort_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ u64 token_key(float x, int index) { return ((u64)sort_key(x + 0.0f) << 32) | (uint32_t)~index; }      // (-0 and 0 are equal)
__device__ __forceinline__ int key_index(u64 k) { return (int)~(uint32_t)k; }

// exp2 in 64 bits: 2^(k / 256) from a table times a polynomial of degree 3 (Taylor, |r| <= 1/512: 1.4e-13), rounded to whole numbers of 2^-44.
struct Weigher {
    double most, c;      // largest logit, log2(e) / T
    const double* table;
    bool infinite;
    __device__ __forceinline__ u64 operator()(float x) const {      // (without branches: several in flight)
        const double d = (double)x - most;
        const double t = fma(d, c, 26388279066624.0);      // 1.5 2^44: to the nearest 256th
        const int k = __double2loint(t);
        const double r = fma(d, c, 26388279066624.0 - t);
        const double q = fma(r, fma(r, fma(r, 0.055504108664821580, 0.24022650695910071), 0.69314718055994531), 1.0);
        const double v = table[k & 255];
        const double w = fma(__hiloint2double(__double2hiint(v) + ((k >> 8) << 20), __double2loint(v)), q, 256.0);      // units of 2^-44
        const u64 whole = t > 26388279066624.0 - 46.0 ? (u64)__double_as_longlong(w) - 0x4070000000000000ull : 0ull;      // (none for -inf and NaN)
        return infinite ? (x == INFINITY ? SF_ONE : 0ull) : whole;
    }
    // bounds on weights in a bin of 64 to a power of two: the rounding of the bin's number (2048 / 64 2^-22 of the exponent) and of exp2 (2^-22) are less than 1e-4 of the exponent
    __device__ __forceinline__ static float above(float b) { return exp2f(fmaf(b, -0.015625f, 44.0001f)) + 1.0f; }
    __device__ __forceinline__ static float below(float b) { return fmaxf(exp2f(fmaf(b, -0.015625f, 43.984275f)) - 1.0f, 0.0f); }
};

struct alignas(16) Shared {      // beside the row and the histogram
    double table[256];
    u64 warp[SF_W], part[SF_CLUSTER];
    u64 cut, total, in_before, sum;
    u64 group[SF_GROUPS], least;
    uint32_t lo[SF_CLUSTER], hi[SF_CLUSTER];
    double dwarp[SF_W];
    int first[2];
    int bin, bin2, upto, inside, n_list, drawn, counts[SF_CLUSTER];
    float drawn_p;
};

template <typename TX>
struct Sampler {
    cg::cluster_group cl = cg::this_cluster();
    const SampleParams& p;
    TX* xs;      // NaN as -inf
    uint32_t* cnt;
    u64* wh;
    Shared* sh;
    int rank, n_cta, warp, lane, base;      // base: token index of xs[0]
    Weigher w;
    float to_bin;
    u64 best;

    __device__ Sampler(const SampleParams& p_) : p(p_) {}

    __device__ __forceinline__ int bin_of(float x) const { return (int)fminf((key_value((uint32_t)(best >> 32)) - x) * to_bin, (float)(SF_BINS - 1)); }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {      // f(value, index) of this warp's tokens that have a value; whole warps
        const TX* x = xs + warp * p.seg;
#pragma unroll 4
        for (int i = lane; i < p.seg; i += 32) f((float)x[i], base + warp * p.seg + i);
    }
    __device__ u64 block_sum(u64 v) const {      // in all threads
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
        __syncthreads();
        if (lane == 0) sh->warp[warp] = v;
        __syncthreads();
        v = 0;
        for (int i = 0; i < SF_W; ++i) v += sh->warp[i];
        return v;
    }
    __device__ u64 cluster_sum(u64 v) {
        v = block_sum(v);
        cl.sync();      // (nobody still reads an earlier sum)
        if (threadIdx.x < n_cta) cl.map_shared_rank(sh, threadIdx.x)->part[rank] = v;
        cl.sync();
        v = 0;
        for (int i = 0; i < n_cta; ++i) v += sh->part[i];
        return v;
    }
    template <typename T>
    __device__ void everywhere(T Shared::* at, T v) {      // (one thread)
        for (int i = 0; i < n_cta; ++i) cl.map_shared_rank(sh, i)->*at = v;
    }
    __device__ int block_last(int v) const {      // the largest, in all threads
        v = __reduce_max_sync(0xffffffffu, v);
        __syncthreads();
        if (lane == 0) sh->warp[warp] = (u64)(v + 1);
        __syncthreads();
        u64 m = 0;
        for (int i = 0; i < SF_W; ++i) m = sh->warp[i] > m ? sh->warp[i] : m;
        return (int)m - 1;
    }
    // inclusive sums of a value a thread, over the CTA
    template <typename V>
    __device__ V scan_in(V v, V* of_warp) const {
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const V o = __shfl_up_sync(0xffffffffu, v, s);
            if (lane >= s) v += o;
        }
        __syncthreads();
        if (lane == 31) of_warp[warp] = v;
        __syncthreads();
        V w = lane < SF_W ? of_warp[lane] : V(0);
#pragma unroll
        for (int s = 1; s < SF_W; s <<= 1) {
            const V o = __shfl_up_sync(0xffffffffu, w, s);
            if (lane >= s) w += o;
        }
        w = __shfl_sync(0xffffffffu, w, warp - 1 & 31);
        return warp ? v + w : v;
    }
    __device__ u64 scan(u64 v) const { return scan_in(v, sh->warp); }
    __device__ double scan(double v) const { return scan_in(v, sh->dwarp); }

    // Numbers per bin of the cluster's tokens, as `fill` counts them in cnt, and the sum of what it returns a thread, in CTA 0's cnt and sum.
    template <typename F>
    __device__ void histogram(F fill) {
        for (int i = threadIdx.x; i < SF_BINS; i += SF_T) cnt[i] = 0;
        if (threadIdx.x == 0) sh->sum = 0;
        cl.sync();      // (CTA 0's are clear before others add to them)
        u64 v = fill();
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
        if (lane == 0 && v) atomicAdd(&cl.map_shared_rank(sh, 0)->sum, v);
        if (rank != 0) {
            __syncthreads();
            for (int b = threadIdx.x; b < SF_BINS; b += SF_T)
                if (cnt[b]) atomicAdd(cl.map_shared_rank(cnt, 0) + b, cnt[b]);
        }
        cl.sync();
    }
    // CTA 0, after histogram(): to everyone, bin = the first bin at which the number of tokens reaches `count` (or the last one with a token), upto = the number of
    // tokens down to and with it, in_before = ahead of it, inside = in it.
    __device__ void find_count(long long count) {
        constexpr int B = SF_BINS / SF_T;
        uint32_t n[B];
        u64 sn = 0;
        int last = -1;      // of the CTA's last bin with a token
        for (int i = 0; i < B; ++i) {
            n[i] = cnt[B * threadIdx.x + i];
            sn += n[i];
            if (n[i]) last = B * (int)threadIdx.x + i;
        }
        u64 an = scan(sn) - sn;
        last = block_last(last);
        for (int i = 0; i < B; ++i) {
            const int b = B * (int)threadIdx.x + i;
            if (((long long)an < count && (long long)(an + n[i]) >= count) || (b == last && (long long)(an + n[i]) < count)) {
                everywhere(&Shared::bin, b);
                everywhere(&Shared::bin2, b);
                everywhere(&Shared::upto, (int)(an + n[i]));
                everywhere(&Shared::inside, (int)n[i]);
                everywhere(&Shared::in_before, an);
            }
            an += n[i];
        }
    }
    // The same for a cut where the weights' sum on top of `before` reaches `goal`, hi(b) and lo(b) bounds on a weight in bin b: bin = the first bin that may reach it,
    // bin2 = the first one that does for sure (or the last one with a token); upto = tokens down to bin2, inside = in bin .. bin2, in_before = ahead of bin.
    template <typename H, typename L>
    __device__ void find_weight(double before, double goal, H hi, L lo) {
        constexpr int B = SF_BINS / SF_T;
        uint32_t n[B];
        double uh = 0.0, ul = 0.0, vh[B], vl[B];
        u64 sn = 0;
        int last = -1;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int b = B * (int)threadIdx.x + i;
            n[i] = cnt[b];
            sn += n[i];
            vh[i] = n[i] ? n[i] * hi(b) : 0.0, vl[i] = n[i] ? n[i] * lo(b) : 0.0;
            uh += vh[i], ul += vl[i];
            if (n[i]) last = b;
        }
        u64 an = scan(sn) - sn;
        double ah = scan(uh) - uh + before, al = scan(ul) - ul + before;
        last = block_last(last);
        const double may = goal * (1.0 - 1e-9), sure = goal * (1.0 + 1e-9);      // (these sums are rounded)
        if (threadIdx.x == 0) sh->first[0] = sh->first[1] = SF_BINS;
        __syncthreads();
        int f[2] = {SF_BINS, SF_BINS};
        double h = ah, l = al;
        for (int i = 0; i < B; ++i) {
            const int b = B * (int)threadIdx.x + i;
            if (!n[i]) continue;
            h += vh[i], l += vl[i];
            if (h >= may && f[0] == SF_BINS) f[0] = b;
            if (l >= sure && f[1] == SF_BINS) f[1] = b;
        }
        for (int i = 0; i < 2; ++i) {
            f[i] = __reduce_min_sync(0xffffffffu, f[i]);
            if (lane == 0 && f[i] < SF_BINS) atomicMin(&sh->first[i], f[i]);
        }
        __syncthreads();
        const int b0 = min(sh->first[0], last), b1 = min(sh->first[1], last);
        for (int i = 0; i < B; ++i) {
            const int b = B * (int)threadIdx.x + i;
            if (b == b0) {
                everywhere(&Shared::bin, b);
                everywhere(&Shared::in_before, an);
            }
            an += n[i];
            if (b == b1) {
                everywhere(&Shared::bin2, b);
                everywhere(&Shared::upto, (int)an);
            }
        }
    }

    // For a cut by weight among the tokens at or above `from`: their number per bin and the sum of their weights (returned), then find_weight().
    __device__ u64 weigh_and_count(u64 from, float per_unit, float top_p) {
        histogram([&]() -> u64 {
            u64 sum = 0;
            if (!from)
                each([&](float x, int) {
                    const u64 v = w(x);
                    if (x > -INFINITY) atomicAdd(cnt + bin_of(x), 1u);
                    sum += v;
                });
            else
                each([&](float x, int i) {
                    if (x > -INFINITY && token_key(x, i) >= from) {
                        atomicAdd(cnt + bin_of(x), 1u);
                        sum += w(x);
                    }
                });
            return sum;
        });
        if (rank == 0) {
            const u64 sum = sh->sum;
            if (threadIdx.x == 0) everywhere(&Shared::total, sum);
            // (bins that are not 64 to a power of two, at extreme temperatures, bound nothing from below)
            const bool bounded = per_unit < 1e30f && !w.infinite;
            find_weight(0.0, (double)top_p * (double)sum, [&](int b) { return bounded ? (double)w.above((float)b) : (double)SF_ONE; },
                        [&](int b) { return bounded && b < SF_BINS - 1 ? (double)w.below((float)b) : 0.0; });
        }
        cl.sync();
        return sh->total;
    }

    // The keys of tokens that `take` names, into CTA 0's list (unordered); its length in CTA 0's n_list, which is 0 before.
    template <typename F>
    __device__ void gather(F take) {
        u64* list = cl.map_shared_rank(wh, 0);
        int* n = &cl.map_shared_rank(sh, 0)->n_list;
        each([&](float x, int i) {
            if (take(x, i)) {
                const int at = atomicAdd(n, 1);
                if (at < SF_LIST) list[at] = token_key(x, i);
            }
        });
        cl.sync();
    }
    __device__ void clear_list() {      // with a meeting of the cluster between it and gather()
        if (rank == 0 && threadIdx.x == 0) sh->n_list = 0;
    }
    // CTA 0: list[0 .. n) sorted, largest first; n <= SF_LIST
    __device__ void sort(u64* list, int n) const {
        int size = 2;
        while (size < n) size <<= 1;
        for (int i = n + threadIdx.x; i < size; i += SF_T) list[i] = 0;
        __syncthreads();
        if (size <= 128) {      // one warp is faster than all of them with barriers
            if (warp == 0)
                for (int k = 2; k <= size; k <<= 1)
                    for (int j = k >> 1; j > 0; j >>= 1) {
                        for (int i = lane; i < size / 2; i += 32) {
                            const int a = 2 * i - (i & (j - 1)), b = a + j;
                            const u64 x = list[a], y = list[b];
                            if ((x < y) == ((a & k) == 0)) list[a] = y, list[b] = x;
                        }
                        __syncwarp();
                    }
            __syncthreads();
            return;
        }
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int i = threadIdx.x; i < size / 2; i += SF_T) {
                    const int a = 2 * i - (i & (j - 1)), b = a + j;
                    const u64 x = list[a], y = list[b];
                    if ((x < y) == ((a & k) == 0)) list[a] = y, list[b] = x;
                }
                __syncthreads();
            }
    }
    // CTA 0: token i of the sorted list's weights ahead of it; two tokens a thread.  pre[0], pre[1]: of tokens 2 t and 2 t + 1; own: theirs
    __device__ void ahead(const u64* list, int n, u64 (&own)[2], u64 (&pre)[2]) const {
        const int t = threadIdx.x;
        own[0] = 2 * t < n ? w(key_value((uint32_t)(list[2 * t] >> 32))) : 0;
        own[1] = 2 * t + 1 < n ? w(key_value((uint32_t)(list[2 * t + 1] >> 32))) : 0;
        pre[0] = scan(own[0] + own[1]) - own[0] - own[1];
        pre[1] = pre[0] + own[0];
    }

    // The key of the last token that a cut by number (count > 0) or by weight keeps, among the tokens at or above `from`, once histogram() and find_*() have
    // run.  total: the sum of their weights, for a cut by weight.  *mine: weights of this thread's tokens that are kept, ahead of the cut's own bin.
    __device__ u64 cut_at(u64 from, long long count, float top_p, u64 total, u64* mine) {
        const bool weights = count <= 0;
        const double goal = (double)top_p * (double)total;
        int b0 = sh->bin, b1 = sh->bin2;
        uint32_t lo = 0, hi = 0xFFFFFFFFu;
        bool by_bin = true;
        auto in = [&](float x, int i) {
            if (!(x > -INFINITY) || (from && token_key(x, i) < from)) return false;
            if (by_bin) {
                const int b = bin_of(x);
                return b >= b0 && b <= b1;
            }
            const uint32_t k = sort_key(x + 0.0f);
            return k >= lo && k <= hi;
        };
        long long kept = (long long)sh->in_before;      // tokens surely kept
        int inside = weights ? sh->upto - (int)kept : sh->inside;
        u64 before = 0;                                 // their weights
        *mine = 0;
        if (weights && b1 > b0 && b1 - b0 < SF_NEAR) {
            // the bounds are few bins apart: the weights of each, a warp's own (its tokens fall into them one by one), then the bin with the cut
            for (int i = threadIdx.x; i < SF_W * SF_NEAR; i += SF_T) wh[i] = 0;
            if (threadIdx.x == 0) sh->sum = 0;
            if (threadIdx.x < SF_NEAR) sh->group[threadIdx.x] = 0;
            cl.sync();
            u64 sum = 0;
            each([&](float x, int i) {
                const int b = x > -INFINITY && (!from || token_key(x, i) >= from) ? bin_of(x) : SF_BINS;
                if (b <= b1) {
                    const u64 v = w(x);
                    if (b < b0) sum += v;
                    else atomicAdd(wh + warp * SF_NEAR + b - b0, v);
                }
            });
            *mine = sum;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            if (lane == 0 && sum) atomicAdd(&cl.map_shared_rank(sh, 0)->sum, sum);
            __syncthreads();
            if (threadIdx.x < SF_NEAR) {
                u64 v = 0;
                for (int i = 0; i < SF_W; ++i) v += wh[i * SF_NEAR + threadIdx.x];
                if (v) atomicAdd(&cl.map_shared_rank(sh, 0)->group[threadIdx.x], v);
            }
            cl.sync();
            if (rank == 0 && threadIdx.x == 0) {
                u64 at = sh->sum;
                u64 tokens = sh->in_before;
                int b = b0;
                for (; b < b1 && (double)(at + sh->group[b - b0]) < goal; ++b) at += sh->group[b - b0], tokens += cnt[b];
                const int n = (int)cnt[b];
                everywhere(&Shared::bin, b);
                everywhere(&Shared::total, at);
                everywhere(&Shared::in_before, tokens);
                everywhere(&Shared::inside, n);
            }
            cl.sync();
            const int b = sh->bin;
            if (lane == 0)
                for (int i = b0; i < b; ++i) *mine += wh[warp * SF_NEAR + i - b0];
            b0 = b1 = b;
            before = sh->total;
            kept = (long long)sh->in_before;
            inside = sh->inside;
            cl.sync();      // (what was written has been read, and the list's place is free)
        } else if (weights) {
            u64 sum = 0;
            each([&](float x, int i) { if (x > -INFINITY && bin_of(x) < b0 && (!from || token_key(x, i) >= from)) sum += w(x); });
            *mine = sum;
            before = cluster_sum(sum);
        }
        for (int round = 0; round < 64; ++round) {      // (each leaves half of 2^32 values at most; equal ones end it)
            if (inside <= SF_LIST) {
                clear_list();
                cl.sync();
                gather(in);
                if (rank == 0) {
                    const int n = min(sh->n_list, SF_LIST);
                    sort(wh, n);
                    u64 own[2], pre[2];
                    ahead(wh, n, own, pre);
                    int last = -1;
                    for (int i = 0; i < 2; ++i) {
                        const int at = 2 * threadIdx.x + i;
                        if (at < n && (weights ? at == 0 || (double)(before + pre[i]) < goal : kept + at < count)) last = at;
                    }
                    last = block_last(last);
                    if (threadIdx.x == 0) everywhere(&Shared::cut, wh[max(last, 0)]);
                }
                cl.sync();
                break;
            }
            // ---- the values' range
            uint32_t a = 0xFFFFFFFFu, z = 0;
            each([&](float x, int i) {
                if (in(x, i)) a = min(a, sort_key(x + 0.0f)), z = max(z, sort_key(x + 0.0f));
            });
            a = __reduce_min_sync(0xffffffffu, a), z = __reduce_max_sync(0xffffffffu, z);
            __syncthreads();
            if (lane == 0) sh->warp[warp] = ((u64)a << 32) | z;
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int i = 0; i < SF_W; ++i) a = min(a, (uint32_t)(sh->warp[i] >> 32)), z = max(z, (uint32_t)sh->warp[i]);
                for (int i = 0; i < n_cta; ++i) cl.map_shared_rank(sh, i)->lo[rank] = a, cl.map_shared_rank(sh, i)->hi[rank] = z;
            }
            cl.sync();
            for (int i = 0; i < n_cta; ++i) a = min(a, sh->lo[i]), z = max(z, sh->hi[i]);
            lo = a, hi = z, by_bin = false;
            if (lo == hi) {      // equal values: so many of them by index
                long long q = count - kept;
                if (weights) {
                    const u64 one = w(key_value(lo));
                    q = one ? (long long)ceil((goal - (double)before) / (double)one) : inside;
                }
                q = min((long long)inside, max(1ll, q));
                int n = 0;
                each([&](float x, int i) { n += in(x, i); });
                n = __reduce_add_sync(0xffffffffu, n);
                __syncthreads();
                if (lane == 0) sh->warp[warp] = n;
                __syncthreads();
                if (threadIdx.x == 0) {
                    int all = 0;
                    for (int i = 0; i < SF_W; ++i) all += (int)sh->warp[i];
                    for (int i = 0; i < n_cta; ++i) cl.map_shared_rank(sh, i)->counts[rank] = all;
                }
                cl.sync();
                long long ahead_of_me = 0;
                for (int i = 0; i < rank; ++i) ahead_of_me += sh->counts[i];
                for (int i = 0; i < warp; ++i) ahead_of_me += (long long)sh->warp[i];
                if (ahead_of_me < q && ahead_of_me + n >= q) {
                    const TX* x = xs + warp * p.seg;
                    for (int i = lane; i < p.seg; i += 32) {
                        const int index = base + warp * p.seg + i;
                        const uint32_t there = __ballot_sync(0xffffffffu, in((float)x[i], index));
                        if (ahead_of_me + __popc(there) >= q) {
                            if ((there >> lane & 1) && ahead_of_me + __popc(there & ((2u << lane) - 1u)) == q) everywhere(&Shared::cut, token_key((float)x[i], index));
                            break;
                        }
                        ahead_of_me += __popc(there);
                    }
                }
                cl.sync();
                break;
            }
            // ---- 2048 parts of that range, falling: keys k with (hi - k) 2048 / width == part
            const u64 width = (u64)hi - lo + 1;
            const uint32_t top = hi;
            auto edge = [&](int part) { return (uint32_t)(((u64)part * width + SF_BINS - 1) / SF_BINS); };      // least top - k of a part
            histogram([&]() -> u64 {
                each([&](float x, int i) {
                    if (in(x, i)) atomicAdd(cnt + (int)((u64)(top - sort_key(x + 0.0f)) * SF_BINS / width), 1u);
                });
                return 0;
            });
            if (rank == 0) {
                if (weights)
                    find_weight((double)before, goal, [&](int b) { return (double)w(key_value(top - edge(b))); }, [&](int b) { return (double)w(key_value(top - (edge(b + 1) - 1))); });
                else
                    find_count(count - kept);
            }
            cl.sync();
            // ---- the bounds' parts; where they are far apart (weights that fall from 1 to 0 within a part), the half of them that has the cut: a round leaves
            // half of the values' range at most
            int p0 = sh->bin, p1 = sh->bin2;
            kept += (long long)sh->in_before;
            inside = sh->upto - (int)sh->in_before;
            cl.sync();      // (what find_*() wrote has been read)
            if (weights) {
                uint32_t above = top - edge(p0);      // keys above it are surely kept
                u64 sum = 0;
                each([&](float x, int i) { if (in(x, i) && sort_key(x + 0.0f) > above) sum += w(x); });
                *mine += sum;
                before += cluster_sum(sum);
                if (p1 - p0 >= SF_BINS / 8) {
                    const int half = (p0 + p1) / 2;
                    const uint32_t mid = top - (edge(half + 1) - 1);      // least key of the upper half
                    int n = 0;
                    sum = 0;
                    each([&](float x, int i) {
                        const uint32_t k = sort_key(x + 0.0f);
                        if (in(x, i) && k <= above && k >= mid) sum += w(x), ++n;
                    });
                    const u64 upper = cluster_sum(sum);
                    const int n_upper = (int)cluster_sum((u64)n);
                    if ((double)(before + upper) >= goal) {
                        p1 = half, inside = n_upper;
                    } else {
                        *mine += sum;
                        before += upper;
                        p0 = half + 1, inside -= n_upper;
                    }
                }
            }
            const uint32_t new_hi = top - edge(p0), new_lo = top - (edge(p1 + 1) - 1);
            hi = new_hi, lo = new_lo;
        }
        const u64 cut = sh->cut;
        if (weights) {
            u64 sum = 0;
            each([&](float x, int i) { if (in(x, i) && token_key(x, i) >= cut) sum += w(x); });
            *mine += sum;
        }
        return cut;
    }

    // Token, its probability and the distribution of the tokens at or above `cut` with weights of `least` at least (the first one always).  mine: the sum of
    // the weights of this thread's kept tokens, if known.
    __device__ void draw(int row, u64 cut, u64 least, float u, const u64* known) {
        auto kept = [&](float x, int i) -> u64 {
            const u64 k = token_key(x, i);
            if (!(x > -INFINITY) || k < cut) return 0ull;
            const u64 v = w(x);
            return v >= least || k == best ? v : 0ull;
        };
        u64 mine = 0;
        if (known) mine = *known;
        else if (!cut && !least) each([&](float x, int) { mine += w(x); });
        else each([&](float x, int i) { mine += kept(x, i); });
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, s);
        cl.sync();      // (nobody still reads an earlier sum)
        if (lane == 0) sh->warp[warp] = mine;
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 v = 0;
            for (int i = 0; i < SF_W; ++i) v += sh->warp[i];
            for (int i = 0; i < n_cta; ++i) cl.map_shared_rank(sh, i)->part[rank] = v;
        }
        cl.sync();
        u64 total = 0, ahead_of_me = 0;
        for (int i = 0; i < n_cta; ++i) {
            if (i < rank) ahead_of_me += sh->part[i];
            total += sh->part[i];
        }
        const u64 goal = goal_of(u, total);
        int drawn = -1;      // in the warp that has it
        float drawn_p = 0.0f;
        if (ahead_of_me <= goal && goal < ahead_of_me + sh->part[rank]) {      // in this CTA: the warp's part that has it is searched by all warps, 32 tokens each in turn
            int found = 0;
            while (found < SF_W - 1 && goal >= ahead_of_me + sh->warp[found]) ahead_of_me += sh->warp[found++];
            const TX* x = xs + found * p.seg;
            const int at = base + found * p.seg, lines = p.seg / 32;
            for (int c = warp; c < lines; c += SF_W) {
                u64 v = kept((float)x[32 * c + lane], at + 32 * c + lane);
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
                if (lane == 0) wh[c] = v;
            }
            __syncthreads();
            if (warp == found) {
                int line = 0;
                while (line < lines - 1 && goal >= ahead_of_me + wh[line]) ahead_of_me += wh[line++];
                const int index = at + 32 * line + lane;
                const u64 own = kept((float)x[32 * line + lane], index);
                u64 v = own;
#pragma unroll
                for (int s = 1; s < 32; s <<= 1) {
                    const u64 o = __shfl_up_sync(0xffffffffu, v, s);
                    if (lane >= s) v += o;
                }
                if (own && ahead_of_me + v - own <= goal && goal < ahead_of_me + v) drawn = index, drawn_p = put(row, index, own, total);
            }
        }
        if (!p.dist) return;
        const int has = __ffs(__ballot_sync(0xffffffffu, drawn >= 0)) - 1;
        if (has >= 0) drawn = __shfl_sync(0xffffffffu, drawn, has), drawn_p = __shfl_sync(0xffffffffu, drawn_p, has);
        distribution(row, cut, least, total, drawn, drawn_p);
    }
    // floor(u total): the draw is the first token up to which the sum is above it
    __device__ static u64 goal_of(float u, u64 total) {
        const float c = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
        return __umul64hi((u64)((double)c * 18446744073709551616.0), total);
    }
    __device__ float put(int row, int index, u64 own, u64 total) const {
        const float f = (float)((double)own / (double)total);
        p.token[row] = index;
        if (p.p) p.p[row] = f;
        return f;
    }
    // Probabilities are f32 results: exp2 in f32, its argument in two terms (2^-22 relative in all); the drawn token's is the one in p.
    __device__ void distribution(int row, u64 cut, u64 least, u64 total, int drawn, float drawn_p) const {
        const float inv = (float)((double)SF_ONE / (double)total), most = (float)w.most, c0 = (float)w.c, c1 = (float)(w.c - (double)c0);
        const uint32_t cut_key = (uint32_t)(cut >> 32);
        float* to = p.dist + (size_t)row * p.V;
        const bool plain = fabsf(c0) < 1e30f && fabsf(most) < 1e30f && c0 > 1e-30f && !w.infinite;
        each([&](float x, int i) {
            if (i >= p.V) return;
            float f = 0.0f;
            const uint32_t k = sort_key(x + 0.0f);
            if (x > -INFINITY && k >= cut_key && (k > cut_key || token_key(x, i) >= cut)) {
                if (plain && least == 0) {
                    // x - most = d + e exactly
                    const float d = x - most, b = d - x, e = (x - (d - b)) + (-most - b), y = d * c0;
                    const float n = rintf(y), z = (y - n) + fmaf(e, c0, fmaf(d, c1, fmaf(d, c0, -y)));
                    float g;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(g) : "f"(z));
                    f = n > -126.0f ? g * inv * __int_as_float(((int)n + 127) << 23) : 0.0f;
                } else {
                    const u64 v = w(x);
                    f = v < least && token_key(x, i) != best ? 0.0f : (float)((double)v / (double)total);
                }
            }
            to[i] = i == drawn ? drawn_p : f;
        });
    }

    // The same as draw_list() for up to 256 tokens: places and sums by comparing each with all.
    __device__ void draw_short(int row, long long count, float top_p, u64 total, u64 least, float u) {
        const int n = sh->n_list, t = threadIdx.x;
        u64 *key = wh, *weight = wh + SF_LIST;
        const u64 mine = t < n ? key[t] : 0, own = t < n ? w(key_value((uint32_t)(mine >> 32))) : 0;
        if (t < n) weight[t] = own;
        if (t == n) key[t] = 0, weight[t] = 0;      // (read in pairs)
        __syncthreads();
        u64 pre = 0;
        int place = 0;
        if (t < n) {
#pragma unroll 2
            for (int j = 0; j < n; j += 2) {
                const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(key + j), v = *reinterpret_cast<const ulonglong2*>(weight + j);
                if (k.x > mine) pre += v.x, ++place;
                if (k.y > mine) pre += v.y, ++place;
            }
            if (count > 0 && place == min((long long)n, count) - 1) sh->total = pre + own;
        }
        __syncthreads();
        if (count > 0) total = sh->total;
        const bool in = t < n && (place == 0 || ((count <= 0 || place < count) && (top_p >= 1.0f || (double)pre < (double)top_p * (double)total) && own >= least));
        const int keep = __syncthreads_count(in);
        if (t < n && place == keep - 1) sh->total = pre + own, sh->cut = mine;
        if (t < n && place >= keep) weight[t] = 0;
        __syncthreads();
        const u64 whole = sh->total, goal = goal_of(u, whole);
        if (in && own) {
            u64 ahead = 0;      // kept ones of lower index: larger low words
#pragma unroll 2
            for (int j = 0; j < n; j += 2) {
                const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(key + j), v = *reinterpret_cast<const ulonglong2*>(weight + j);
                if ((uint32_t)k.x > (uint32_t)mine) ahead += v.x;
                if ((uint32_t)k.y > (uint32_t)mine) ahead += v.y;
            }
            if (ahead <= goal && goal < ahead + own) {
                sh->drawn = key_index(mine);
                sh->drawn_p = put(row, sh->drawn, own, whole);
            }
        }
        __syncthreads();
    }

    // CTA 0's sorted list holds all tokens down to the cut by number, or by weight of `total`: the filters and the draw.
    __device__ void draw_list(int row, long long count, float top_p, u64 total, u64 least, float u) {
        u64* list = wh;
        u64* other = wh + SF_LIST;
        const int n = min(sh->n_list, SF_LIST), t = threadIdx.x;
        sort(list, n);
        u64 own[2], pre[2];
        ahead(list, n, own, pre);
        if (count > 0) {      // the first `count` are the whole
            const u64 in = (2 * t < count ? own[0] : 0) + (2 * t + 1 < count ? own[1] : 0);
            total = block_sum(in);
        }
        const double goal = (double)top_p * (double)total;
        int last = 0;
        for (int i = 0; i < 2; ++i) {
            const int at = 2 * t + i;
            if (at < n && (count <= 0 || at < count) && (top_p >= 1.0f || (double)pre[i] < goal) && own[i] >= least) last = at;
        }
        const int keep = block_last(last) + 1;
        const u64 whole = block_sum((2 * t < keep ? own[0] : 0) + (2 * t + 1 < keep ? own[1] : 0));
        if (t == 0) sh->cut = list[keep - 1], sh->total = whole;
        // the kept ones by rising index: largest first of (~index, place)
        for (int i = t; i < keep; i += SF_T) other[i] = ((u64)(uint32_t)list[i] << 32) | (uint32_t)i;
        sort(other, keep);
        for (int i = 0; i < 2; ++i) own[i] = 2 * t + i < keep ? w(key_value((uint32_t)(list[(uint32_t)other[2 * t + i]] >> 32))) : 0;
        const u64 upto = scan(own[0] + own[1]), target = goal_of(u, whole);
        u64 a = upto - own[0] - own[1];
        for (int i = 0; i < 2; ++i) {
            if (own[i] && a <= target && target < a + own[i]) {
                sh->drawn = (int)~(uint32_t)(other[2 * t + i] >> 32);
                sh->drawn_p = put(row, sh->drawn, own[i], whole);
            }
            a += own[i];
        }
        __syncthreads();
    }
};

template <typename TX>
__global__ void __launch_bounds__(SF_T, 2) k_sample_filter(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Sampler<TX> s(p);
    s.rank = (int)s.cl.block_rank(), s.n_cta = (int)s.cl.num_blocks(), s.warp = threadIdx.x >> 5, s.lane = threadIdx.x & 31;
    s.wh = reinterpret_cast<u64*>(smem);
    s.cnt = reinterpret_cast<uint32_t*>(s.wh + SF_BINS);
    s.sh = reinterpret_cast<Shared*>(s.cnt + SF_BINS);
    s.xs = reinterpret_cast<TX*>(s.sh + 1);
    s.base = s.rank * SF_W * p.seg;
    const int row = blockIdx.x / s.n_cta;
    for (int i = threadIdx.x; i < 256; i += SF_T) s.sh->table[i] = exp2((double)i * 0.00390625);
    pdl_wait();
    pdl_launch_dependents();
    // ---- the row's part, NaN as -inf; its largest token
    const TX* src = reinterpret_cast<const TX*>(p.logits) + (size_t)row * p.ld;
    u64 best = 0;
    {
        TX* x = s.xs + s.warp * p.seg;
        const int at0 = s.base + s.warp * p.seg;
        float top = -INFINITY;
        int top_at = 0;
        auto take = [&](float v, int i) {
            if (!(v > -INFINITY)) v = -INFINITY;
            if (v > top) top = v, top_at = at0 + i;      // (a lane's tokens come by rising index)
            return v;
        };
        constexpr int PER = 16 / sizeof(TX), IN_FLIGHT = 4;
        if (((uintptr_t)(src + at0) & 15) == 0) {
            for (int i0 = s.lane * PER; i0 < p.seg; i0 += IN_FLIGHT * 32 * PER) {
                struct alignas(16) Piece {      // taken and stored as sixteen bytes
                    TX x[PER];
                } v[IN_FLIGHT];
                static_assert(sizeof(v) == 16 * IN_FLIGHT && alignof(Piece) == 16, "pieces are loads of 16 bytes");
#pragma unroll
                for (int c = 0; c < IN_FLIGHT; ++c) {
                    const int i = i0 + c * 32 * PER;
                    if (i < p.seg && at0 + i + PER <= p.V) *reinterpret_cast<uint4*>(v[c].x) = __ldg(reinterpret_cast<const uint4*>(src + at0 + i));
                }
#pragma unroll
                for (int c = 0; c < IN_FLIGHT; ++c) {
                    const int i = i0 + c * 32 * PER;
                    if (i >= p.seg) break;
                    float f[PER];
                    if (at0 + i + PER <= p.V) {
#pragma unroll
                        for (int j = 0; j < PER; ++j) f[j] = take((float)v[c].x[j], i + j);
                    } else {
#pragma unroll
                        for (int j = 0; j < PER; ++j) f[j] = take(at0 + i + j < p.V ? (float)src[at0 + i + j] : -INFINITY, i + j);
                    }
#pragma unroll
                    for (int j = 0; j < PER; ++j) v[c].x[j] = (TX)f[j];
                    *reinterpret_cast<uint4*>(x + i) = *reinterpret_cast<const uint4*>(v[c].x);
                }
            }
        } else {
#pragma unroll 4
            for (int i = s.lane; i < p.seg; i += 32) x[i] = (TX)take(at0 + i < p.V ? (float)src[at0 + i] : -INFINITY, i);
        }
        if (top > -INFINITY) best = token_key(top, top_at);
    }
    // ---- the largest token of each of 256 groups of threads, in all CTAs
    const int lanes = 2 * s.n_cta, per_cta = SF_GROUPS / s.n_cta;
    for (int k = 1; k < lanes; k <<= 1) {
        const u64 o = __shfl_xor_sync(0xffffffffu, best, k);
        best = o > best ? o : best;
    }
    if (s.lane % lanes == 0) {
        const int g = s.rank * per_cta + threadIdx.x / lanes;
        for (int i = 0; i < s.n_cta; ++i) s.cl.map_shared_rank(s.sh, i)->group[g] = best;
    }
    s.clear_list();
    if (threadIdx.x == 0) s.sh->least = 0;
    s.cl.sync();
    best = 0;
#pragma unroll
    for (int i = 0; i < SF_GROUPS / 32; ++i) best = s.sh->group[s.lane + 32 * i] > best ? s.sh->group[s.lane + 32 * i] : best;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
        const u64 o = __shfl_xor_sync(0xffffffffu, best, k);
        best = o > best ? o : best;
    }
    s.best = best;
    const float T = p.temperature ? p.temperature[row] : 1.0f, top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f, u = p.u[row];
    const int top_k = p.top_k ? p.top_k[row] : 0;
    if (best == 0) {      // no token has a weight
        if (s.rank == 0 && threadIdx.x == 0) {
            p.token[row] = -1;
            if (p.p) p.p[row] = 0.0f;
        }
        if (p.dist)
            s.each([&](float, int i) { if (i < p.V) p.dist[(size_t)row * p.V + i] = 0.0f; });
        s.cl.sync();
        return;
    }
    const float most = key_value((uint32_t)(best >> 32));
    s.w.most = (double)most, s.w.c = 1.4426950408889634 / (double)T, s.w.table = s.sh->table, s.w.infinite = most == INFINITY;
    const long long count = top_k > 0 && top_k < p.V ? top_k : 0;
    const bool by_weight = top_p < 1.0f;
    const u64 least = min_p > 0.0f ? (u64)ceil((double)fminf(min_p, 1.0f) * (double)SF_ONE) : 0ull;
    if (!(T > 0.0f) || count == 1 || top_p <= 0.0f || min_p > 1.0f) {      // the first token alone
        if (s.rank == 0 && threadIdx.x == 0) s.put(row, key_index(best), 1, 1);
        if (p.dist) s.each([&](float x, int i) { if (i < p.V) p.dist[(size_t)row * p.V + i] = token_key(x, i) == best && x > -INFINITY ? 1.0f : 0.0f; });
        s.cl.sync();
        return;
    }
    if (!count && !by_weight) {
        s.draw(row, 0, least, u, nullptr);
        s.cl.sync();
        return;
    }
    // bins: 64 to a unit of the logits where the cut goes by number, 64 to a power of two of the weights where it goes by weight
    const float weight_bins = s.w.infinite ? 0.0f : fminf(64.0f * 1.44269504f / T, 1e30f);
    s.to_bin = s.w.infinite ? 0.0f : count ? 64.0f : weight_bins;
    u64 total = 0;
    bool listed = false;
    if (count) {
        if (count <= SF_GROUPS * 3 / 4) {
            // `count` groups have a token at or above the count-th largest of the groups' largest ones: so lie the first `count` tokens
            const u64 mine = s.sh->group[threadIdx.x % SF_GROUPS];
            int place = 0;
            if (threadIdx.x < SF_GROUPS) {
#pragma unroll 8
                for (int j = 0; j < SF_GROUPS; j += 2) {
                    const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(s.sh->group + j);
                    place += (k.x > mine) + (k.y > mine);
                }
                if (place == count - 1 && mine) s.sh->least = mine;      // (groups without a token are 0)
            }
            __syncthreads();
            const u64 from = s.sh->least;
            if (from) {
                s.gather([&](float x, int i) { return x > -INFINITY && token_key(x, i) >= from; });
                listed = *s.cl.map_shared_rank(&s.sh->n_list, 0) <= SF_LIST;
                s.cl.sync();
            }
        }
        if (!listed) {
            s.clear_list();
            s.histogram([&]() -> u64 {
                s.each([&](float x, int) { if (x > -INFINITY) atomicAdd(s.cnt + s.bin_of(x), 1u); });
                return 0;
            });
            if (s.rank == 0) s.find_count(count);
            s.cl.sync();
        }
    } else {
        total = s.weigh_and_count(0, weight_bins, top_p);
    }
    if (!listed && s.sh->upto <= SF_LIST) {
        const int bin = s.sh->bin2;
        s.gather([&](float x, int) { return x > -INFINITY && s.bin_of(x) <= bin; });
        listed = true;
    }
    if (listed) {
        if (s.rank == 0) {
            if (s.sh->n_list <= SF_SHORT) s.draw_short(row, count, top_p, total, least, u);
            else s.draw_list(row, count, top_p, total, least, u);
        }
        if (p.dist) {
            if (s.rank == 0 && threadIdx.x == 0) {
                const Shared& z = *s.sh;
                s.everywhere(&Shared::cut, z.cut);
                s.everywhere(&Shared::total, z.total);
                s.everywhere(&Shared::drawn, z.drawn);
                s.everywhere(&Shared::drawn_p, z.drawn_p);
            }
            s.cl.sync();
            s.distribution(row, s.sh->cut, 0, s.sh->total, s.sh->drawn, s.sh->drawn_p);
        }
        return;
    }
    u64 cut = 0, mine = 0;
    if (count) {
        cut = s.cut_at(0, count, 1.0f, 0, &mine);
        if (by_weight) {
            s.cl.sync();
            s.to_bin = weight_bins;
            total = s.weigh_and_count(cut, weight_bins, top_p);
            cut = s.cut_at(cut, 0, top_p, total, &mine);
        }
    } else {
        cut = s.cut_at(0, 0, top_p, total, &mine);
    }
    s.draw(row, cut, least, u, by_weight && least == 0 ? &mine : nullptr);
    s.cl.sync();
}

size_t sample_smem(int seg, size_t type) { return SF_BINS * 12 + sizeof(Shared) + (size_t)SF_W * seg * type; }

template <typename TX>
int launch_sample(dc_ctx* ctx, SampleParams p, int rows) {
    auto seg_of = [&](int n) { return ((p.V + n * SF_W - 1) / (n * SF_W) + 31) / 32 * 32; };
    // few CTAs a row (fewer meetings), but two of them fit into an SM, and all SMs have work as long as a CTA has 4096 tokens
    int n = 1;
    while (n < 8 && sample_smem(seg_of(n), sizeof(TX)) > 112 * 1024) n *= 2;
    while (n < SF_CLUSTER && rows * n * 2 <= ctx->num_sms && p.V / n > 4096) n *= 2;
    p.seg = seg_of(n);
    const size_t smem = sample_smem(p.seg, sizeof(TX));
    DC_TRY(dc_kernel_setup(ctx, (const void*)k_sample_filter<TX>, (int)sample_smem(SF_MOST / SF_W, 4), "k_sample_filter"));
    if (n > 8) DC_TRY(dc_check_cuda(ctx, cudaFuncSetAttribute((const void*)k_sample_filter<TX>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "k_sample_filter"));
    return dc_launch_cluster(ctx, "k_sample_filter", k_sample_filter<TX>, dim3(rows * n), dim3(SF_T), smem, n, p);
}

}  // namespace

extern "C" {

int dc_b200_sample_rows_dev(dc_ctx* ctx, const void* logits_dev, int type, int rows, int vocab, int64_t ld, const float* temperature_dev, const int32_t* top_k_dev,
                            const float* top_p_dev, const float* min_p_dev, const float* uniforms_dev, int32_t* tokens_dev, float* p_dev, float* dist_dev) {
    if (!ctx) return DC_B200_INVALID_ARGUMENT;
    if (ld == 0) ld = vocab;
    if (rows < 0 || vocab < 1 || ld < vocab) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "sample_rows: bad shape (%d rows of %d, stride %lld)", rows, vocab, (long long)ld);
    if (type != DC_TYPE_F32 && type != DC_TYPE_BF16) return dc_fail(ctx, DC_B200_UNSUPPORTED, "sample_rows: logits of type %d (F32 and BF16 are supported)", type);
    if (vocab > SF_VOCAB || rows > (1 << 20)) return dc_fail(ctx, DC_B200_UNSUPPORTED, "sample_rows: %d rows of %d tokens", rows, vocab);
    if (rows == 0) return DC_B200_OK;
    if (!logits_dev || !uniforms_dev || !tokens_dev) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "sample_rows: null buffer");
    cudaSetDevice(ctx->device);
    SampleParams p = {logits_dev, (size_t)ld, vocab, 0, temperature_dev, top_k_dev, top_p_dev, min_p_dev, uniforms_dev, tokens_dev, p_dev, dist_dev};
    return type == DC_TYPE_F32 ? launch_sample<float>(ctx, p, rows) : launch_sample<__nv_bfloat16>(ctx, p, rows);
}

int dc_b200_sample_rows(dc_ctx* ctx, const float* logits_host, int rows, int vocab, const float* temperature, const int32_t* top_k, const float* top_p,
                        const float* min_p, const float* uniforms, int32_t* tokens_out, float* p_out, float* dist_out) {
    if (!ctx) return DC_B200_INVALID_ARGUMENT;
    if (!logits_host || !uniforms || !tokens_out || rows < 1 || vocab < 1) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "sample_rows: bad argument");
    for (int i = 0; i < rows; ++i)
        if (!(uniforms[i] >= 0.0f && uniforms[i] < 1.0f) || (temperature && !(temperature[i] >= 0.0f)) || (top_p && !(top_p[i] > 0.0f)) || (min_p && !(min_p[i] >= 0.0f && min_p[i] <= 1.0f)) ||
            (top_k && top_k[i] < 0))
            return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "sample_rows: row %d has a setting out of range", i);
    cudaSetDevice(ctx->device);
    const size_t big = (size_t)rows * vocab * 4, small = ((size_t)rows * 4 + 255) / 256 * 256, pad = (big + 255) / 256 * 256;
    uint8_t* s = dc_scratch(ctx, pad * (dist_out ? 2 : 1) + 7 * small);
    if (!s) return DC_B200_OUT_OF_MEMORY;
    float* l = (float*)s;
    uint8_t* at = s + pad + (dist_out ? pad : 0);
    auto up = [&](const void* from) -> uint8_t* {      // (pageable sources: the copy is done with them when it returns)
        uint8_t* to = at;
        at += small;
        if (from && cudaMemcpyAsync(to, from, (size_t)rows * 4, cudaMemcpyHostToDevice, ctx->stream) != cudaSuccess) return nullptr;
        return from ? to : nullptr;
    };
    DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(l, logits_host, big, cudaMemcpyHostToDevice, ctx->stream), "sample_rows"));
    uint8_t *dt = up(temperature), *dk = up(top_k), *dp = up(top_p), *dm = up(min_p), *du = up(uniforms), *tok = at, *pr = at + small;
    DC_TRY(dc_check_cuda(ctx, cudaGetLastError(), "sample_rows"));
    DC_TRY(dc_b200_sample_rows_dev(ctx, l, DC_TYPE_F32, rows, vocab, 0, (float*)dt, (int32_t*)dk, (float*)dp, (float*)dm, (float*)du, (int32_t*)tok, (float*)pr,
                                   dist_out ? (float*)(s + pad) : nullptr));
    auto down = [&](void* to, const void* from, size_t n) { return to ? dc_check_cuda(ctx, cudaMemcpyAsync(to, from, n, cudaMemcpyDeviceToHost, ctx->stream), "sample_rows") : DC_B200_OK; };
    DC_TRY(down(tokens_out, tok, (size_t)rows * 4));
    DC_TRY(down(p_out, pr, (size_t)rows * 4));
    DC_TRY(down(dist_out, s + pad, big));
    return dc_b200_synchronize(ctx);
}

}  // extern "C"
