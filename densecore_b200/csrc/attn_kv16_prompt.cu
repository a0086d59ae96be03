// Attention of prompt-sized portions over the paged cache of 16-bit rows whose sequences are kept on the GPU, on the 5th-generation tensor cores.
//
// One CTA per (256 rows of a sequence, key head, part of the keys): row r is new token r / G and query head r % G of the key head, so that any number of query heads a
// key head fills the tiles.  Two sets of 128 rows share key and value tiles of 64 keys (four pages, copied as they lie: the cache holds them in the operands'
// swizzles).  Scores and P V are tcgen05.mma with f32 accumulators in tensor memory: per set two tiles of scores of 64 columns, whose first 32 then hold the
// weights as pairs of the cache's type, and HD columns of answers; the next tile's scores are made while a thread per row weights this one's.
//   warps 0-7    weights: four a set, thread = row = tensor-memory lane
//   warp 8       copies pages
//   warps 9-10   issue a set's products each
//   warp 11      looks over the values of tiles that not all rows see all of
// Weights are rounded to the cache's type (bf16 2^-9, fp16 2^-12) and summed as rounded, so that a row's answer is an average of its values: an error like that of the result's own
// rounding, of a sum of many.  fp16 ends at 2^-25: the reference of a row's weights lies 2^14 below its maximum where it is taken anew and follows from 2^15 on, so that what is lost is below 2^-39 of the
// of the largest (from 2^7 on it took 56 us for a prompt of 2011 tokens for 60 now, and a row whose answer is the rest's beside a key 22 natural units ahead was off by three times its rounding).
// Answers are the tensor cores' f32 sums, which are cut off by some 2^-23 of themselves an instruction, always towards 0: 150000 keys of one CTA leave a row 1e-3 too small (2000 leave it 1.4e-5), which is
// a quarter of bf16's rounding and twice fp16's.
// A value that is infinite or NaN in a tile of which some row does not see all enters it as 0, or the products would carry it to rows that do not see it; rows that do see
// it are NaN in that dimension.
// Keys are split over CTAs where there are fewer tiles of rows than SMs; the rows kernel, which follows, adds the parts up (the last CTA of a tile alone took 160 us over a kernel of 30).
// Bound: the chain of a tile, scores, weights, answers, some 1900 cycles with the exponentials' pipe at 38 % and the issue slots at 39 %, and a CTA's start, whose queries come from HBM: 2011 tokens,
// bf16, 32 / 4 heads of 128: 33 GFLOP in 54 us, 617 TFLOP/s, 252 CTAs on 148 SMs.  512 tokens behind 6001 with a window of 2048 and 3 single tokens, 16 / 8 heads: 50 us.
// Sixteen warps of weights, two threads a row: 69 for 70 us at the time, for the pairs' barriers.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_kv16_tiles.cuh"
#include "dc_launch.cuh"
#include "dc_tcgen05.cuh"

using namespace dc;

#define DC_TRY(expr)                       \
    do {                                   \
        int _st = (expr);                  \
        if (_st != DC_B200_OK) return _st; \
    } while (0)

namespace {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
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
template <typename TC>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    if constexpr (std::is_same<TC, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename TC>
__device__ __forceinline__ float2 unpack(uint32_t w) {
    if constexpr (std::is_same<TC, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
// K-major rows of 32 bytes with the 32-byte swizzle (8-row groups of 256 bytes, chunk c of row r at place c ^ (r >> 2 & 1))
__device__ __forceinline__ uint64_t umma_desc_sw32(uint32_t saddr) {
    const uint32_t lo = ((saddr >> 4) & 0x3FFFu) | (1u << 16), hi = (256u >> 4) | (1u << 14) | (6u << 29);
    return ((uint64_t)hi << 32) | lo;
}

struct PromptParams {
    const dc_kv_entry* entries;
    const int32_t *numbers, *tables;
    int pages_per_seq, slots, heads, n_kv, least, num_sms;      // least: sequences of more rows than this
    const void* q;
    int64_t ldq, ldo;
    const uint8_t* arena;
    float scale;
    int window, keep;
    void* out;
    float* parts;
};

constexpr int KP_KEYS = 64, KP_STAGES = 4, KP_THREADS = 12 * 32;
enum KpBar { KP_FULL = 0, KP_PRE = 4, KP_FREE = 8, KP_S = 12, KP_P = 16, KP_O = 20, KP_DRAIN = 22, KP_QUERY = 24, KP_NBARS = 25 };
template <int HD>
struct Lay {
    static constexpr uint32_t SET = KP_ROWS * HD * 2, TILE = KP_KEYS * HD * 2;      // a set's queries: halves of 64 columns; keys or values of a tile
    static constexpr uint32_t KV = 2 * SET, BAD = KV + KP_STAGES * 2 * TILE, SICK = BAD + KP_STAGES * HD * 8, BARS = SICK + 2 * KP_ROWS * HD / 8;
    static constexpr size_t SMEM = BARS + KP_NBARS * 8 + 1024;
};
template <int HD, typename TC>
__global__ void __launch_bounds__(KP_THREADS, 1) k_kv16_prompt(const PromptParams p, int* err) {
    using L = Lay<HD>;
    using R = dc_kv16_rec<HD>;
    constexpr bool F16 = std::is_same<TC, __half>::value;
    // (a half that is infinite or NaN has an exponent of ones: its top bit in (w & EXPONENTS) + ONE)
    constexpr uint32_t EXPONENTS = F16 ? 0x7C007C00u : 0x7F807F80u, ONE = F16 ? 0x04000400u : 0x00800080u, TOPS = 0x80008000u;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_bad[KP_STAGES];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, kvh = blockIdx.x % p.n_kv, item = blockIdx.x / p.n_kv, G = p.heads / p.n_kv;
    pdl_wait();
    // ---- the item: which tile of rows, and which part of its keys
    const TileLine tiles(p.entries, p.numbers + DC_KV_ENTRIES, p.slots, G, p.least, p.n_kv, p.num_sms);
    if (blockIdx.x == 0 && tid == 0 && (long long)tiles.n_all * p.n_kv > gridDim.x) atomicExch(err, DC_ERR_STEP);      // (a step of more than the launch was made for)
    const int line = item / tiles.most, part = item % tiles.most;
    if (line >= tiles.n_all) return;
    const Tile tl(tiles, line, p.window, p.keep);
    if (part >= tl.n_parts) return;
    const dc_kv_entry own = tl.e;
    const int row0 = tl.row0, rows = tl.rows, sets = rows > KP_ROWS ? 2 : 1, first = tl.first, last = tl.last, window = p.window ? min(p.window, 0x40000000) : 0x40000000 /* positions are below 2^30 */, n_pages = tl.pages.n, n_parts = tl.n_parts, kept = tl.pages.kept, low = tl.pages.low;
    const int tile0 = (int)((long long)tl.key_tiles * part / n_parts), n_tiles = (int)((long long)tl.key_tiles * (part + 1) / n_parts) - tile0;
    auto page_at = [&](int i) { return tl.pages.at(i); };
    // position of the first key of page i of tile t; far behind the last token where there is none
    auto key_at = [&](int t, int i) { return 4 * (tile0 + t) + i < n_pages ? page_at(4 * (tile0 + t) + i) * DC_KV_BLOCK : 0x40000000; };
    // Tiles that tokens at positions least .. greatest see all of: a run of them, of those that have no kept page
    struct Run {
        int from;
        uint32_t n;
        __device__ __forceinline__ bool operator()(int t) const { return (uint32_t)(t - from) < n; }
    };
    auto run_of = [&](int least, int greatest) -> Run {
        const int seen_from = max(tl.pages.low * DC_KV_BLOCK, greatest - window + 1), pages_to = min((least + 1) / DC_KV_BLOCK, n_pages - kept + low);      // the first key, the first page behind
        const int page_from = (seen_from + DC_KV_BLOCK - 1) / DC_KV_BLOCK, from = max(0, (page_from - low + kept + 3) / 4 - tile0), to = (pages_to - low + kept) / 4 - tile0;
        return {from, (uint32_t)max(0, to - from)};
    };
    const Run whole = run_of(first, last);
    const uint32_t sm = (smem_u32(smem) + 1023u) & ~1023u;
    uint8_t* const base = smem + (sm - smem_u32(smem));
    auto bar = [sm](int which, int i = 0) -> uint32_t { return sm + L::BARS + 8u * (uint32_t)(which + i); };
    if (warp == 9) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < KP_NBARS; ++i) mbar_init(bar(i), i == KP_QUERY ? sets * KP_ROWS : i >= KP_FREE && i < KP_S ? sets : i >= KP_P && i < KP_O ? 4 : 1);
        mbar_fence_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();      // (not before the tensor memory is there: a successor that held some and waited for this kernel would never give it back)
    const uint32_t tmem = s_tmem;
    auto wait = [&](uint32_t b, uint32_t parity) {      // (a role that gives up lets the others run into limits of their own)
        const bool is = mbar_wait_warp(b, parity);
        if (!is && err) atomicExch(err, DC_ERR_MBAR_TIMEOUT);
        return is;
    };
    if (warp < 8) {
        // ------------------------------------------------------------------ weights
        const int u = warp >> 2, row = 32 * (warp & 3) + lane, r = KP_ROWS * u + row;
        if (u < sets) {
            const uint32_t t_unit = tmem + u * 256 + ((uint32_t)(32 * (warp & 3)) << 16), t_o = t_unit + 128;
            const int warp_row = row0 + KP_ROWS * u + 32 * (warp & 3), n_own = own.count * G - warp_row;      // the warp's first row, rows from there on
            const int my_token = min((row0 + r) / G, own.count - 1), qp = own.pos0 + my_token;
            const int w_first = own.pos0 + min(warp_row / G, own.count - 1), w_last = own.pos0 + min((warp_row + 31) / G, own.count - 1);
            const Run whole_here = run_of(w_first, w_last);
            // ---- the warp's queries, neighbouring lanes along a row; negated where the scale is negative
            const uint32_t area = sm + u * L::SET + 32 * (warp & 3) * 128;      // the warp's 32 rows; after the last product they hold its results
            constexpr int LANES = HD / 8, PER = 32 / LANES, ROUNDS = 32 / PER;      // lanes of a row, rows at a time, times
            const int c8 = lane % LANES;
            auto row_at = [&](int i) { return PER * i + lane / LANES; };        // (of the warp's 32)
            auto place = [&](int rr, int c) { return area + (c >> 3) * (KP_ROWS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4); };
            // the lane's rows in turn: where token and head of each lie in rows of queries or results
            struct Walk {
                int j, g;
            };
            const Walk walk0 = {(warp_row + lane / LANES) / G, (warp_row + lane / LANES) % G};
            auto on = [&](Walk& x) {
                x.g += PER;
                while (x.g >= G) x.g -= G, ++x.j;      // (once at most, but for G < PER)
            };
            auto element = [&](const Walk& x, int64_t ld) { return (size_t)(own.tok0 + x.j) * ld + (size_t)(kvh * G + x.g) * HD + 8 * c8; };
            const int n_rows = min(n_own, rows - KP_ROWS * u - 32 * (warp & 3));      // rows that there are, of the warp's 32
            {
                const uint32_t sign = p.scale < 0.0f ? 0x80008000u : 0u;
                uint4 v[ROUNDS];      // (all on their way at once)
                Walk x = walk0;
#pragma unroll
                for (int i = 0; i < ROUNDS; ++i) {
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (row_at(i) < n_rows) {
                        const uint16_t* at = reinterpret_cast<const uint16_t*>(p.q) + element(x, p.ldq);
                        if (((uintptr_t)at & 15) == 0) v[i] = __ldg(reinterpret_cast<const uint4*>(at));
                        else v[i] = make_uint4(at[0] | (uint32_t)at[1] << 16, at[2] | (uint32_t)at[3] << 16, at[4] | (uint32_t)at[5] << 16, at[6] | (uint32_t)at[7] << 16);
                    }
                    on(x);
                }
#pragma unroll
                for (int i = 0; i < ROUNDS; ++i) sts128(place(row_at(i), c8), v[i].x ^ sign, v[i].y ^ sign, v[i].z ^ sign, v[i].w ^ sign);
            }
            uint32_t* sick = reinterpret_cast<uint32_t*>(base + L::SICK) + r * (HD / 32);      // the row's dimensions that have met a value that is no number
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) sick[i] = 0;
            fence_async_smem();
            mbar_arrive(bar(KP_QUERY));
            __syncwarp();
            const float sl2 = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-45f);      // (above 0, if only the least there is: minus infinity stays so)
            // A row's largest weight where its reference is taken anew, and how far the maximum goes ahead until it is, in powers of two: fp16 ends at 2^16
            constexpr float LARGEST = F16 ? 14.0f : 0.0f, LAG = F16 ? 1.0f : 8.0f;
            static_assert(!F16 || LARGEST + LAG <= 15.0f, "weights are fp16 numbers");
            float m_run = -3e38f, l_run[2] = {0.0f, 0.0f};
            bool ok = true;
            __syncwarp();
            {
                const uint32_t zero[16] = {};
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) tmem_st16(t_o + 16 * c, zero);      // (complete and ordered with the first tile's weights)
            }
            for (int t = 0; t < n_tiles; ++t) {
                const uint32_t t_s = t_unit + 64 * (t & 1);
                ok = wait(bar(KP_S, 2 * u + (t & 1)), (t >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const bool masked = !whole_here(t);
                uint32_t seen[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};      // the tile's keys that the row sees
                if (!whole(t)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k0 = key_at(t, i);
                        auto below = [](int n) { return (1u << min(max(n, 0), 16)) - 1u; };      // the page's first n keys
                        const uint32_t is = below(qp + 1 - k0) & (~below(qp + 1 - window - k0) | below(p.keep - k0)) & 0xFFFFu;
                        seen[i >> 1] = i & 1 ? (seen[i >> 1] & 0xFFFFu) | is << 16 : (seen[i >> 1] & 0xFFFF0000u) | is;
                    }
                }
                int x[4][16] = {};
                auto s = [&](int i) -> float { return __int_as_float(x[i >> 4][i & 15]); };
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld16(t_s + 16 * i, x[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld_wait(x[i]);
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (!(seen[i >> 5] >> (i & 31) & 1u)) x[i >> 4][i & 15] = __float_as_int(-INFINITY);
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], s(i));
                if (!whole(t)) {      // (as warp 11 goes by)
                    const int stage = t % KP_STAGES;
                    ok = wait(bar(KP_FULL, stage), (t / KP_STAGES) & 1);
                    if (!ok) break;
                    if (s_bad[stage]) {
                        const uint2* bad = reinterpret_cast<const uint2*>(base + L::BAD) + stage * HD;
#pragma unroll 1
                        for (int d = 0; d < HD; ++d)
                            if ((bad[d].x & seen[0]) | (bad[d].y & seen[1])) sick[d >> 5] |= 1u << (d & 31);
                    }
                    __syncwarp();
                }
                const float m_new = fmaxf(m_run, fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), sl2, -LARGEST));
                // the reference follows once the largest score is 2^LAG further above it: weights up to there are as exact, and the answers' factors are rare
                if (__any_sync(0xffffffffu, m_new > m_run + LAG)) {
                    const float corr = ex2(m_run - m_new);
                    m_run = m_new;
#pragma unroll
                    for (int i = 0; i < 2; ++i) l_run[i] *= corr;
                    if (t > 0) {
                        ok = wait(bar(KP_O, u), (t - 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD / 16; ++c) {
                            int o[16];
                            uint32_t w[16];
                            tmem_ld16(t_o + 16 * c, o);
                            tmem_ld_wait(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__int_as_float(o[i]) * corr);
                            tmem_st16(t_o + 16 * c, w);
                        }
                    }
                }
                const uint64_t sl2_2 = pair(sl2, sl2), m_2 = pair(-m_run, -m_run);
                uint64_t l_2[2] = {pair(l_run[0], l_run[1]), 0};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 y = unpair(fma2(pair(s(32 * h + 2 * i), s(32 * h + 2 * i + 1)), sl2_2, m_2));
                        w[i] = pack<TC>(ex2(y.x), ex2(y.y));
                        const float2 f = unpack<TC>(w[i]);
                        l_2[i & 1] = add2(l_2[i & 1], pair(f.x, f.y));
                    }
                    __syncwarp();      // masks are a lane's own, stores are the whole warp's
                    tmem_st16(t_s + 16 * h, w);      // (columns whose scores have been read)
                }
                {
                    const float2 f = unpair(add2(l_2[0], l_2[1]));
                    l_run[0] = f.x, l_run[1] = f.y;
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(KP_P, 2 * u + (t & 1)));      // (two barriers: a warp may be done with the next tile before another is with this one)
            }
            if (ok) ok = wait(bar(KP_DRAIN, u), 0);      // (a barrier of its own: of two phases of the tiles' one, both of which may be complete, the first cannot be told from the next)
            if (ok) {
                tc_fence_after();
                const float l = l_run[0] + l_run[1];
                auto factor = [&](int c, int i, float mul) { return sick[(16 * c + i) >> 5] >> ((16 * c + i) & 31) & 1 ? NAN : mul; };
                bool any_sick = false;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) any_sick = any_sick || sick[i];
                // rows by way of shared memory, so that neighbouring lanes store along a row; f32 parts 64 dimensions at a time
                if (n_parts == 1) {
                    const float mul = 1.0f / l;
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        int o[16];
                        __syncwarp();
                        tmem_ld16(t_o + 16 * c, o);
                        tmem_ld_wait(o);
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = pack<TC>(__int_as_float(o[2 * i]) * mul, __int_as_float(o[2 * i + 1]) * mul);
                        if (any_sick) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) w[i] = pack<TC>(__int_as_float(o[2 * i]) * factor(c, 2 * i, mul), __int_as_float(o[2 * i + 1]) * factor(c, 2 * i + 1, mul));
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) sts128(place(lane, 2 * c + i), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    }
                    __syncwarp();
                    uint4 v[ROUNDS];
#pragma unroll
                    for (int i = 0; i < ROUNDS; ++i) v[i] = lds128(place(row_at(i), c8));
                    Walk x = walk0;
#pragma unroll
                    for (int i = 0; i < ROUNDS; ++i) {
                        if (row_at(i) < n_rows) {
                            uint16_t* at = reinterpret_cast<uint16_t*>(p.out) + element(x, p.ldo);
                            if (((uintptr_t)at & 15) == 0) {
                                *reinterpret_cast<uint4*>(at) = v[i];
                            } else {
                                const uint4 f = v[i];
                                at[0] = f.x & 0xFFFF, at[1] = f.x >> 16, at[2] = f.y & 0xFFFF, at[3] = f.y >> 16, at[4] = f.z & 0xFFFF, at[5] = f.z >> 16, at[6] = f.w & 0xFFFF, at[7] = f.w >> 16;
                            }
                        }
                        on(x);
                    }
                } else {
                    float* to = p.parts + ((size_t)(line * tiles.most + part) * p.n_kv + kvh) * kp_part_floats<HD>() + (KP_ROWS * u + 32 * (warp & 3)) * (HD + 4);
                    if (lane < n_rows) *reinterpret_cast<float2*>(to + (size_t)lane * (HD + 4) + HD) = make_float2(m_run, l);
                    constexpr int LN = HD == 128 ? 16 : 8;      // lanes of a row: 64 dimensions of four bytes, or 32
#pragma unroll 1
                    for (int g = 0; g < HD / (4 * LN); ++g) {
#pragma unroll 1
                        for (int c = 0; c < LN / 4; ++c) {
                            int o[16];
                            __syncwarp();
                            tmem_ld16(t_o + 4 * LN * g + 16 * c, o);
                            tmem_ld_wait(o);
                            if (any_sick) {
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_int(__int_as_float(o[i]) * factor(LN / 4 * g + c, i, 1.0f));
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) sts128(place(lane, 4 * c + i), o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                        __syncwarp();
#pragma unroll 4
                        for (int i = 0; i < ROUNDS; ++i) {
                            const int rr = row_at(i);
                            const uint4 v = lds128(place(rr, c8));
                            if (rr < n_rows) *reinterpret_cast<uint4*>(to + (size_t)rr * (HD + 4) + 4 * LN * g + 4 * c8) = v;
                        }
                    }
                }
            }
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------------ pages: lanes 0-3 one each of a tile (behind the last: the last, which nobody sees there)
        const int32_t* table = p.tables + (size_t)own.seq * p.pages_per_seq;
        int page = 0;
        auto look_up = [&](int t) {
            if (lane < 4 && t < n_tiles) page = table[page_at(min(4 * (tile0 + t) + lane, n_pages - 1))];
        };
        look_up(0);
        uint32_t uses = 0;      // of the stages' first barriers, odd or even
        int t = 0;
        for (; t < n_tiles; ++t) {
            const int stage = t % KP_STAGES;
            if (t >= KP_STAGES && !wait(bar(KP_FREE, stage), (t / KP_STAGES - 1) & 1)) break;
            uses ^= whole(t) ? 0u : 1u << stage;
            const uint32_t b = whole(t) ? bar(KP_FULL, stage) : bar(KP_PRE, stage);
            if (lane == 0) mbar_expect_tx(b, 2 * L::TILE);
            __syncwarp();
            if (lane < 4) {
                const uint8_t* from = p.arena + ((size_t)page * p.n_kv + kvh) * R::BYTES;
                const uint32_t to = sm + L::KV + stage * (2 * L::TILE) + lane * R::VALUES;
                bulk_g2s(to, from, R::VALUES, b);
                bulk_g2s(to + L::TILE, from + R::VALUES, R::VALUES, b);
            }
            look_up(t + 1);
        }
        // no copy may still be in flight when the CTA leaves (at once unless someone gave up)
        for (int i = max(0, t - KP_STAGES); i < t; ++i) {
            const int stage = i % KP_STAGES;
            if (whole(i)) mbar_wait_warp(bar(KP_FULL, stage), (i / KP_STAGES) & 1);
            else mbar_wait_warp(bar(KP_PRE, stage), ~(uses >> stage) & 1);
        }
    } else if (warp == 11) {
        // ------------------------------------------------------------------ values of tiles that not all rows see all of
        uint32_t uses = 0;      // of the stages' first barriers, odd or even
        for (int t = 0; t < n_tiles; ++t) {
            if (whole(t)) continue;
            const int stage = t % KP_STAGES;
            if (!wait(bar(KP_PRE, stage), uses >> stage & 1)) break;
            uses ^= 1u << stage;
            const uint32_t values = sm + L::KV + stage * (2 * L::TILE) + L::TILE;
            uint32_t tops = 0;
#pragma unroll 8
            for (int i = lane; i < (int)L::TILE / 16; i += 32) {
                const uint4 v = lds128(values + 16 * i);
                tops |= ((v.x & EXPONENTS) + ONE) | ((v.y & EXPONENTS) + ONE) | ((v.z & EXPONENTS) + ONE) | ((v.w & EXPONENTS) + ONE);
            }
            const bool odd = __any_sync(0xffffffffu, tops & TOPS);
            if (odd) {      // which keys, by dimension; and 0 in their place
                uint32_t* bad = reinterpret_cast<uint32_t*>(base + L::BAD) + stage * HD * 2;
                for (int i = lane; i < 2 * HD; i += 32) bad[i] = 0;
                __syncwarp();
#pragma unroll 1
                for (int i = lane; i < (int)L::TILE / 16; i += 32) {
                    const uint4 v = lds128(values + 16 * i);
                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    const int d = (i >> 1) % HD, key = (i >> 1) / HD * 16 + 8 * ((i & 1) ^ ((d >> 2) & 1));
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t is = __vcmpeq2(w[c] & EXPONENTS, EXPONENTS);
                        w[c] &= ~is;
                        const uint32_t two = (is & 1u) | (is >> 15 & 2u);
                        if (two) atomicOr(bad + 2 * d + ((key + 2 * c) >> 5), two << ((key + 2 * c) & 31));
                    }
                    sts128(values + 16 * i, w[0], w[1], w[2], w[3]);
                }
            }
            if (lane == 0) s_bad[stage] = odd;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(KP_FULL, stage));
        }
    } else if (warp - 9 < sets) {
        // ------------------------------------------------------------------ products
        const int u = warp - 9;
        const bool one = elect_one();
        constexpr uint32_t id_s = F16 ? umma_idesc_f16(KP_ROWS, KP_KEYS) : umma_idesc_bf16(KP_ROWS, KP_KEYS), id_o = F16 ? umma_idesc_f16(KP_ROWS, HD) : umma_idesc_bf16(KP_ROWS, HD);
        const uint64_t q = umma_desc_sw128(sm + u * L::SET, 1024), dk = umma_desc_sw128(sm + L::KV, R::GROUP), dv = umma_desc_sw32(sm + L::KV + L::TILE);
        const uint32_t t_unit = tmem + u * 256;
        auto scores = [&](int t) {
            if (one) {
                const uint64_t k = dk + (t % KP_STAGES) * (2 * L::TILE / 16);
                const uint32_t d = t_unit + 64 * (t & 1);
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) umma_f16(d, q + ((i >> 2) * (KP_ROWS * 128) + 32 * (i & 3)) / 16, k + ((i >> 2) * 1024 + 32 * (i & 3)) / 16, id_s, i > 0);
                umma_commit(bar(KP_S, 2 * u + (t & 1)));
            }
        };
        auto values = [&](int t) {
            if (one) {
                const uint64_t v = dv + (t % KP_STAGES) * (2 * L::TILE / 16);
                const uint32_t w = t_unit + 64 * (t & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) umma_f16_ts(t_unit + 128, w + 8 * i, v + i * (R::VALUES / 16), id_o, 1);
                umma_commit(bar(KP_O, u));
                if (t == n_tiles - 1) umma_commit(bar(KP_DRAIN, u));
                umma_commit(bar(KP_FREE, t % KP_STAGES));
            }
        };
        bool ok = wait(bar(KP_QUERY), 0) && wait(bar(KP_FULL, 0), 0);
        if (ok) {
            tc_fence_after();
            scores(0);
        }
        // scores of tile t + 1 go where the weights of tile t - 1 were, once the product that reads those is complete; ahead of the wait for tile t's weights
        for (int t = 0; t < n_tiles && ok; ++t) {
            if (t + 1 < n_tiles) {
                ok = wait(bar(KP_FULL, (t + 1) % KP_STAGES), ((t + 1) / KP_STAGES) & 1);
                if (ok && t > 0) ok = wait(bar(KP_O, u), (t - 1) & 1);
                tc_fence_after();
                if (ok) scores(t + 1);
            }
            ok = ok && wait(bar(KP_P, 2 * u + (t & 1)), (t >> 1) & 1);
            tc_fence_after();
            if (ok) values(t);
        }
        if (!ok) {      // products in flight still read shared and tensor memory
            if (one) umma_commit(bar(KP_DRAIN, u));
            mbar_wait_warp(bar(KP_DRAIN, u), 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

template <int HD, typename TC>
int launch(dc_ctx* ctx, const PromptParams& p, int items) {
    DC_TRY(dc_kernel_setup_unspilled(ctx, (const void*)k_kv16_prompt<HD, TC>, (int)Lay<HD>::SMEM, "k_kv16_prompt"));
    return dc_launch(ctx, "k_kv16_prompt", k_kv16_prompt<HD, TC>, dim3(items * p.n_kv), dim3(KP_THREADS), Lay<HD>::SMEM, p, ctx->d_err);
}

}  // namespace

// Parts: as many as CTAs where keys are split (a tile that is not split has none).
size_t dc_kv16_prompt_parts(int num_sms, int n_kv, int dim) { return (size_t)std::max(1, num_sms / n_kv) * n_kv * KP_TILE_ROWS * (dim + 4) * 4; }

int dc_launch_kv16_prompt(dc_ctx* ctx, const dc_kv16_call& c) {
    const dc_kv_dev& z = *c.kv->dev;
    const long long G = z.heads / z.kv, tokens = std::min((long long)z.max_tokens, (long long)z.slots * z.max_count);
    // tiles: at most one that is not full for every sequence with that many new tokens
    const long long least = dc_kv16_rows(z.type) / G + 1, tiles = tokens * G / KP_TILE_ROWS + std::min((long long)z.slots, tokens / least);
    const int items = (int)std::max(tiles, (long long)std::max(1, ctx->num_sms / z.kv));
    const PromptParams p = {z.entries, z.numbers, z.tables, z.pages_per_seq, z.slots, z.heads, z.kv, dc_kv16_rows(z.type), ctx->num_sms, c.q, c.ldq, c.ldo, c.arena, c.scale, c.window, c.keep, c.out,
                            z.prompt_parts};
    if (z.type == DC_TYPE_F16) return z.dim == 128 ? launch<128, __half>(ctx, p, items) : launch<64, __half>(ctx, p, items);
    return z.dim == 128 ? launch<128, __nv_bfloat16>(ctx, p, items) : launch<64, __nv_bfloat16>(ctx, p, items);
}
