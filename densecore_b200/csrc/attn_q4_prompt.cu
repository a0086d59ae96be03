// Attention of prompt-sized portions over the cache in 4 bits, bf16 rows, on the 5th-generation tensor cores.
//
// One CTA per (256 rows of an entry, key head, part of the keys): row r is new token r / G and query head r % G of the key head, so that any number of query heads a key
// head fills the tiles.  Two sets of 128 rows share key and value tiles of 64 keys.  Scores and P V are tcgen05.mma with f32 accumulators in tensor memory: per
// set two tiles of scores of 64 columns, whose first 32 then hold the weights as fp16 pairs, and HD columns of answers; the next tile's scores are made while a
// thread per row weights this one's.
//   warps 0-7    weights: four a set, thread = row = tensor-memory lane
//   warps 8-15   pages by bulk copies, codes turned into fp16 rows of the operands' 128-byte swizzle (d c + m, rounded once: 2^-11 relative); a warp has the keys
//                or the values of one page, values turned (rows are dimensions: products with keys along the rows took three times as long to issue)
//   warps 16-17  issue a set's products each (one warp for both was the bound: some 50 cycles a product)
// Queries are bf16 rows times a power of two (exact in fp16), weights fp16 (2^-11, the largest at 2^7: down to 2^-32 of it), keys and
// values fp32(d c + m) rounded to fp16 (2^-11): together below a bf16 result's own 2^-8.
// A value that is not a number (d = m = NaN) enters the tiles as 0, or the products would carry it to rows that do not see it; the CTA keeps the first
// position of such a value per group of 64 dimensions, and rows that see it end as NaN there.
// Bound: the weights' arithmetic and the chain scores, weights, answers of a tile, one CTA per SM: 2011 tokens, 32 query heads, 4 key heads of 128: 59.3 us, 559 TFLOP/s; the
// matrix pipe is busy for 28 % of the time, issue slots for 54 %.  Steps on the way: table entries read once a page, not one load after the other, and rows of queries and results
// stored coalesced; two issuing warps; references that follow rarely.
// Keys are split over CTAs where there are fewer row tiles than SMs (dc_q4_tiles); k_q4_join adds the parts up.
#include <math.h>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_launch.cuh"
#include "dc_q4.h"
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
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ __half2 as_h2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
// two codes in the halves' low four bits, anything above: d c + m
__device__ __forceinline__ uint32_t value2(uint32_t w, __half2 d, __half2 m) {
    const __half2 v = __hfma2(__hadd2(as_h2((w & 0x000F000Fu) | 0x64006400u), __floats2half2_rn(-1024.0f, -1024.0f)), d, m);      // 1024 + c - 1024
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Four words 16 bytes apart, from lanes whose places differ by 64 bytes: each lane starts at another one of the four, so that the lanes meet in no bank.
__device__ __forceinline__ void lds_turned(uint32_t at, int turn, uint32_t (&w)[4]) {
    uint32_t x[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = lds32(at + ((c + turn) & 3) * 16);
    const bool odd = turn & 1, two = turn & 2;
    const uint32_t y0 = odd ? x[3] : x[0], y1 = odd ? x[0] : x[1], y2 = odd ? x[1] : x[2], y3 = odd ? x[2] : x[3];
    w[0] = two ? y2 : y0, w[1] = two ? y3 : y1, w[2] = two ? y0 : y2, w[3] = two ? y1 : y3;
}

struct PromptParams {
    const dc_q4_tile* tiles;
    const int32_t* joins;
    float* ws;
    const __nv_bfloat16* q;
    int ldq, ldo, heads, n_kv, max_blocks;
    const int32_t* tables;
    const uint8_t* arena;
    float scale;
    __nv_bfloat16* out;
};

constexpr int QP_ROWS = 128, QP_KEYS = 64, QP_STAGES = 4, QP_RAW = 3, QP_THREADS = 18 * 32;
enum QpBar { QP_FULL = 0, QP_FREE = 4, QP_S = 8, QP_P = 12, QP_O = 16, QP_DRAIN = 18, QP_PAGES = 20, QP_READ = 23, QP_QUERY = 26, QP_NBARS = 27 };
template <int HD>
struct Lay {
    static constexpr uint32_t SET = QP_ROWS * HD * 2, TILE = QP_KEYS * HD * 2;      // a set's queries; keys or values of a tile: halves of 64 columns
    static constexpr uint32_t KV = 2 * SET, RAW = KV + QP_STAGES * 2 * TILE, RAW_BYTES = 4 * dc_q4_rec<HD>::BYTES, BARS = RAW + QP_RAW * RAW_BYTES;
    static constexpr size_t SMEM = BARS + QP_NBARS * 8 + 1024;
};

template <int HD>
__global__ void __launch_bounds__(QP_THREADS, 1) k_q4_prompt(const PromptParams p, int* err) {
    using L = Lay<HD>;
    using R = dc_q4_rec<HD>;
    constexpr int GR = R::GROUPS;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_nan[2];
    __shared__ float s_pow[2 * QP_ROWS];      // 2^e of a row
    pdl_wait();
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, kvh = blockIdx.x % p.n_kv, tile = blockIdx.x / p.n_kv, G = p.heads / p.n_kv;
    const dc_q4_tile* tp = p.tiles + tile;
    const dc_q4_tile tl = *tp;
    const int rows = min(2 * QP_ROWS, tl.count * G - tl.row0), sets = rows > QP_ROWS ? 2 : 1;
    const int last = tl.pos0 + (tl.row0 + rows - 1) / G, first_tile = tl.tile0, n_tiles = tl.tile1 - tl.tile0;
    const uint32_t sm = (smem_u32(smem) + 1023u) & ~1023u;
    auto bar = [sm](int which, int i = 0) -> uint32_t { return sm + L::BARS + 8u * (uint32_t)(which + i); };
    if (warp == 16) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < QP_NBARS; ++i) mbar_init(bar(i), i == QP_QUERY ? sets * QP_ROWS : i >= QP_FREE && i < QP_S ? sets : i < QP_FREE || i >= QP_READ ? 256 : i >= QP_P && i < QP_O ? 4 : 1);
        mbar_fence_init();
        s_nan[0] = s_nan[1] = 0x7fffffff;
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
        const int u = warp >> 2, row = 32 * (warp & 3) + lane, r = QP_ROWS * u + row;
        if (u < sets) {
            const uint32_t t_unit = tmem + u * 256 + ((uint32_t)(32 * (warp & 3)) << 16), t_o = t_unit + 128;
            const bool in = r < rows;
            auto token = [&](const dc_q4_tile& z) { return (z.row0 + r) / G; };
            const int my_token = token(tl);
            const int qp = in ? tl.pos0 + my_token : -1, all_see = tl.pos0 + (tl.row0 + QP_ROWS * u + 32 * (warp & 3)) / G;
            // ---- the warp's queries, neighbouring lanes along a row: a row times 2^-e, 2^e <= its largest < 2^(e + 1)
            const uint32_t own = sm + u * L::SET + 32 * (warp & 3) * 128;      // the warp's 32 rows; after the last product they hold its results
            constexpr int LANES = HD / 8, PER = 32 / LANES, BATCH = 4;          // lanes of a row, rows at a time
            const int c8 = lane % LANES;
            auto row_at = [&](int i) { return PER * i + lane / LANES; };       // (of the warp's 32)
            auto place = [&](int rr, int c) { return own + (c >> 3) * (QP_ROWS * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4); };
            // the lane's own row: its token and head; a row's first element in rows of queries or results, from the lane that has it (whole warps)
            auto element = [&](const dc_q4_tile& z, int j, int rr, int ld) {
                const int jr = __shfl_sync(0xffffffffu, j, rr), g = z.row0 + QP_ROWS * u + 32 * (warp & 3) + rr - jr * G;
                return (size_t)(z.tok0 + jr) * ld + (size_t)(kvh * G + g) * HD;
            };
            const int n_first = rows - (QP_ROWS * u + 32 * (warp & 3));          // rows that there are, of the warp's 32
            auto f2 = [](uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); };
#pragma unroll 1
            for (int i0 = 0; i0 < 32 / PER; i0 += BATCH) {
                uint4 v[BATCH];
                float most[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int rr = row_at(i0 + i);
                    const __nv_bfloat16* src = p.q + element(tl, my_token, rr, p.ldq) + 8 * c8;
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (rr < n_first) {
                        if (((uintptr_t)src & 15) == 0) {
                            v[i] = __ldg(reinterpret_cast<const uint4*>(src));
                        } else {
                            const uint16_t* at = reinterpret_cast<const uint16_t*>(src);
                            v[i] = make_uint4(at[0] | (uint32_t)at[1] << 16, at[2] | (uint32_t)at[3] << 16, at[4] | (uint32_t)at[5] << 16, at[6] | (uint32_t)at[7] << 16);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                    most[i] = 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) most[i] = fmaxf(most[i], fmaxf(fabsf(f2(w[k]).x), fabsf(f2(w[k]).y)));
                }
#pragma unroll
                for (int k = 1; k < LANES; k <<= 1)
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], k));
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int rr = row_at(i0 + i), e = max(-100, min(100, (int)(__float_as_uint(most[i]) >> 23) - 127));
                    const float up = __uint_as_float((uint32_t)(127 - e) << 23) * (p.scale < 0.0f ? -1.0f : 1.0f);
                    auto half = [&](uint32_t x) { return pack_h2(f2(x).x * up, f2(x).y * up); };
                    sts128(place(rr, c8), half(v[i].x), half(v[i].y), half(v[i].z), half(v[i].w));
                    if (c8 == 0) s_pow[QP_ROWS * u + 32 * (warp & 3) + rr] = __uint_as_float((uint32_t)(127 + e) << 23);
                }
            }
            fence_async_smem();
            mbar_arrive(bar(QP_QUERY));
            __syncwarp();
            const float sl2 = fmaxf(fabsf(p.scale) * 1.4426950408889634f * s_pow[r], 1e-35f);      // (above 0: minus infinity stays so)
            float m_run = -1e30f, l_run[2] = {0.0f, 0.0f};
            bool ok = true;
            __syncwarp();
            {
                const uint32_t zero[16] = {};
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) tmem_st16(t_o + 16 * c, zero);      // (complete and ordered with the first tile's weights)
            }
            for (int t = 0; t < n_tiles; ++t) {
                const uint32_t t_s = t_unit + 64 * (t & 1);
                ok = wait(bar(QP_S, 2 * u + (t & 1)), (t >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const int k0 = (first_tile + t) * QP_KEYS;
                const bool masked = k0 + QP_KEYS - 1 > all_see;
                int x[2][16] = {};      // 32 scores at a time, once for their largest and once for the weights: all 64 would not stay in registers
                auto s = [&](int i) -> float { return __int_as_float(x[i >> 4][i & 15]); };
                auto load = [&](int h) {
                    tmem_ld16(t_s + 32 * h, x[0]);
                    tmem_ld16(t_s + 32 * h + 16, x[1]);
                    tmem_ld_wait(x[0]);
                    tmem_ld_wait(x[1]);
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (k0 + 32 * h + i > qp) x[i >> 4][i & 15] = __float_as_int(-INFINITY);
                    }
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __syncwarp();
                    load(h);
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], s(i));
                }
                const float m_new = fmaxf(m_run, fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), sl2, -7.0f));
                // the largest weight is 2^7, so that the others keep fp16's range down to 2^-32 of it: where its value is next to nothing, they are the answer.  The
                // reference follows once the largest score is 2^8 above it: weights up to 2^15 are as exact, and the answers' factors are rare
                if (__any_sync(0xffffffffu, m_new > m_run + 8.0f)) {
                    const float corr = ex2(m_run - m_new);
                    m_run = m_new;
#pragma unroll
                    for (int i = 0; i < 2; ++i) l_run[i] *= corr;
                    if (t > 0) {
                        ok = wait(bar(QP_O, u), (t - 1) & 1);
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
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
                    __syncwarp();      // masks are a lane's own, loads and stores are the whole warp's
                    load(h);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float a = ex2(fmaf(s(2 * i), sl2, -m_run)), b = ex2(fmaf(s(2 * i + 1), sl2, -m_run));
                        l_run[i & 1] += a + b;
                        w[i] = pack_h2(a, b);
                    }
                    __syncwarp();
                    tmem_st16(t_s + 16 * h, w);      // (columns whose scores have been read)
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(QP_P, 2 * u + (t & 1)));      // (two barriers: a warp may be done with the next tile before another is with this one)
            }
            // (phase by phase: the parity of the last alone also stands for the one before the last but one; tile t's scores come behind phase t - 2)
            if (ok && n_tiles > 1) ok = wait(bar(QP_O, u), (n_tiles - 2) & 1);
            if (ok) ok = wait(bar(QP_O, u), (n_tiles - 1) & 1);
            if (ok) {
                tc_fence_after();
                const float l = l_run[0] + l_run[1];
                const dc_q4_tile te = *tp;      // (again: what stays in registers meanwhile spills)
                const bool whole = te.n_splits == 1;
                const int n_own = te.count * G - te.row0 - (QP_ROWS * u + 32 * (warp & 3));
                const float mul = 1.0f / l;
                // rows by way of shared memory, so that neighbouring lanes store along a row; f32 parts 64 dimensions at a time
                if (whole) {
#pragma unroll 1
                    for (int c = 0; c < HD / 16; ++c) {
                        int o[16];
                        __syncwarp();
                        tmem_ld16(t_o + 16 * c, o);
                        tmem_ld_wait(o);
                        const float f = s_nan[c / 4] <= qp ? NAN : mul;
                        auto v = [&](int i) { return __int_as_float(o[i]) * f; };
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            sts128(place(lane, 2 * c + i), pack_bf2(v(8 * i), v(8 * i + 1)), pack_bf2(v(8 * i + 2), v(8 * i + 3)), pack_bf2(v(8 * i + 4), v(8 * i + 5)), pack_bf2(v(8 * i + 6), v(8 * i + 7)));
                    }
                    __syncwarp();
                    const int own_token = token(te);
#pragma unroll 8
                    for (int i = 0; i < 32 / PER; ++i) {
                        const int rr = row_at(i);
                        __nv_bfloat16* dst = p.out + element(te, own_token, rr, p.ldo) + 8 * c8;
                        const uint4 v = lds128(place(rr, c8));
                        if (rr >= n_own) continue;
                        if (((uintptr_t)dst & 15) == 0) {
                            *reinterpret_cast<uint4*>(dst) = v;
                        } else {
                            uint16_t* at = reinterpret_cast<uint16_t*>(dst);
                            at[0] = v.x & 0xFFFF, at[1] = v.x >> 16, at[2] = v.y & 0xFFFF, at[3] = v.y >> 16, at[4] = v.z & 0xFFFF, at[5] = v.z >> 16, at[6] = v.w & 0xFFFF, at[7] = v.w >> 16;
                        }
                    }
                } else {
                    float* part = p.ws + (((size_t)te.ws * p.n_kv + (size_t)te.n_splits * kvh + te.split) * (2 * QP_ROWS) + QP_ROWS * u + 32 * (warp & 3)) * (HD + 4);
                    if (in) *reinterpret_cast<float2*>(part + (size_t)lane * (HD + 4) + HD) = make_float2(m_run, l);
                    constexpr int LN = HD == 128 ? 16 : 8;      // lanes of a row: 64 dimensions of four bytes, or 32
#pragma unroll 1
                    for (int g = 0; g < HD / (4 * LN); ++g) {
#pragma unroll 1
                        for (int c = 0; c < LN / 4; ++c) {
                            int o[16];
                            __syncwarp();
                            tmem_ld16(t_o + 4 * LN * g + 16 * c, o);
                            tmem_ld_wait(o);
                            const float f = s_nan[(4 * LN * g + 16 * c) / 64] <= qp ? NAN : 1.0f;
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                sts128(place(lane, 4 * c + i), __float_as_uint(__int_as_float(o[4 * i]) * f), __float_as_uint(__int_as_float(o[4 * i + 1]) * f),
                                       __float_as_uint(__int_as_float(o[4 * i + 2]) * f), __float_as_uint(__int_as_float(o[4 * i + 3]) * f));
                        }
                        __syncwarp();
#pragma unroll 4
                        for (int i = 0; i < 32 / PER; ++i) {
                            const int rr = row_at(i);
                            const uint4 v = lds128(place(rr, c8));
                            if (rr < n_own) *reinterpret_cast<uint4*>(part + (size_t)rr * (HD + 4) + 4 * LN * g + 4 * c8) = v;
                        }
                    }
                }
            }
        }
    } else if (warp < 16) {
        // ------------------------------------------------------------------ key and value tiles
        const int lw = warp & 3;      // a warp has one page
        const int32_t* table = p.tables + (size_t)tl.seq * p.max_blocks;
        const int last_page = last / DC_KV_BLOCK;
        // warp 8, lanes 0-3: a page each of a tile (those beyond the last token: the last page, for something finite); the block of the next fetch is read ahead
        int fetched = 0, t = 0, block = 0;
        auto look_up = [&](int t) {
            if (lane < 4 && t < n_tiles) block = table[min((first_tile + t) * 4 + lane, last_page)];
        };
        auto fetch = [&] {
            const uint32_t b = bar(QP_PAGES, fetched % QP_RAW);
            if (lane == 0) mbar_expect_tx(b, L::RAW_BYTES);
            __syncwarp();
            if (lane < 4)
                bulk_g2s(sm + L::RAW + (fetched % QP_RAW) * L::RAW_BYTES + lane * R::BYTES, p.arena + ((size_t)block * p.n_kv + kvh) * R::BYTES, R::BYTES, b);
            look_up(++fetched);
        };
        if (warp == 8) {
            look_up(0);
            while (fetched < QP_RAW && fetched < n_tiles) fetch();
        }
        for (; t < n_tiles; ++t) {
            bool ok = wait(bar(QP_PAGES, t % QP_RAW), (t / QP_RAW) & 1);
            if (ok && t >= QP_STAGES) ok = wait(bar(QP_FREE, t % QP_STAGES), (t / QP_STAGES - 1) & 1);
            if (!ok) break;
            const uint32_t to = sm + L::KV + (t % QP_STAGES) * (2 * L::TILE);
            const uint32_t raw = sm + L::RAW + (t % QP_RAW) * L::RAW_BYTES + lw * R::BYTES;
            const int pos = (first_tile + t) * QP_KEYS + lw * DC_KV_BLOCK;
            if (warp < 12) {
                // ---- keys: rows of the operand are tokens; a lane takes 32 dimensions of one token at a time
                constexpr int N = HD / 64;
                uint32_t w[N][4], sc[N];
                const int i = HD == 128 ? lane >> 3 : lane >> 4;
#pragma unroll
                for (int x = 0; x < N; ++x) {      // (all loads ahead of the stores, which they may not pass)
                    const int tok = HD == 128 ? (lane & 7) + 8 * x : lane & 15;
                    sc[x] = lds32(raw + R::K_SCALES + (tok * GR + i / 2) * 4);
                    lds_turned(raw + R::k_word(tok, 0, i), (tok & 7) >> 1, w[x]);
                }
#pragma unroll
                for (int x = 0; x < N; ++x) {
                    const int tok = HD == 128 ? (lane & 7) + 8 * x : lane & 15, key = lw * 16 + tok;
                    const __half2 dm = as_h2(sc[x]), d = __low2half2(dm), m = __high2half2(dm);
                    const uint32_t at = to + (i >> 1) * (QP_KEYS * 128) + key * 128;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        sts128(at + (((4 * (i & 1) + c) ^ (key & 7)) << 4), value2(w[x][0] >> (4 * c), d, m), value2(w[x][1] >> (4 * c), d, m), value2(w[x][2] >> (4 * c), d, m),
                               value2(w[x][3] >> (4 * c), d, m));
                }
            } else {
                // ---- values: rows of the operand are dimensions; a lane takes the page's 16 tokens of two dimensions, 8 apart, at a time
                const uint32_t scales = raw + R::V_SCALES;
                if (lane < 16 * GR) {      // what is not a number or beyond the last token is 0
                    const int tok = lane / GR;
                    const bool nan = (lds32(scales + 4 * lane) & 0x7FFFu) > 0x7C00u;
                    if (pos + tok > last || nan) {
                        if (nan && pos + tok <= last) atomicMin(&s_nan[lane % GR], pos + tok);
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(scales + 4 * lane), "r"(0) : "memory");
                    }
                }
                __syncwarp();
                constexpr int N = HD / 64;
                const int d8 = lane & 7;
                uint32_t w[N][4], sc[16 * GR];
#pragma unroll
                for (int x = 0; x < N; ++x) lds_turned(raw + (R::v_byte(0, d8, (lane >> 3) + 4 * x)), d8 >> 1, w[x]);
#pragma unroll
                for (int x = 0; x < 16 * GR / 4; ++x) {
                    const uint4 f = lds128(scales + 16 * x);
                    sc[4 * x] = f.x, sc[4 * x + 1] = f.y, sc[4 * x + 2] = f.z, sc[4 * x + 3] = f.w;
                }
#pragma unroll
                for (int x = 0; x < N; ++x)
#pragma unroll
                    for (int a = 0; a < 2; ++a) {      // tokens 8 a .. 8 a + 7
                        __half2 d[4], m[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t u = sc[(8 * a + 2 * c) * GR + x], v = sc[(8 * a + 2 * c + 1) * GR + x];
                            d[c] = as_h2(__byte_perm(u, v, 0x5410)), m[c] = as_h2(__byte_perm(u, v, 0x7632));
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int dim = 16 * ((lane >> 3) + 4 * x) + 8 * h + d8, sh = 8 * a + 4 * h;
                            sts128(to + L::TILE + dim * 128 + (((2 * lw + a) ^ d8) << 4), value2(w[x][0] >> sh, d[0], m[0]), value2(w[x][1] >> sh, d[1], m[1]), value2(w[x][2] >> sh, d[2], m[2]),
                                   value2(w[x][3] >> sh, d[3], m[3]));
                        }
                    }
            }
            fence_async_smem();
            mbar_arrive(bar(QP_FULL, t % QP_STAGES));
            mbar_arrive(bar(QP_READ, t % QP_RAW));
            if (warp == 8 && t + QP_RAW < n_tiles) {      // the pages' place is free once all have read them
                if (!wait(bar(QP_READ, t % QP_RAW), (t / QP_RAW) & 1)) break;
                fetch();
            }
        }
        if (warp == 8 && lane == 0)
            for (; t < fetched; ++t) mbar_wait(bar(QP_PAGES, t % QP_RAW), (t / QP_RAW) & 1, nullptr);      // (given up: copies in flight)
    } else if (warp - 16 < sets) {
        // ------------------------------------------------------------------ products
        const int u = warp - 16;
        const bool one = elect_one();
        constexpr uint32_t id_s = umma_idesc_f16(QP_ROWS, QP_KEYS), id_o = umma_idesc_f16(QP_ROWS, HD);
        const uint64_t q = umma_desc_sw128(sm + u * L::SET, 1024), dk = umma_desc_sw128(sm + L::KV, 1024), dv = umma_desc_sw128(sm + L::KV + L::TILE, 1024);
        const uint32_t t_unit = tmem + u * 256;
        auto scores = [&](int t) {
            if (one) {
                const uint64_t k = dk + (t % QP_STAGES) * (2 * L::TILE / 16);
                const uint32_t d = t_unit + 64 * (t & 1);
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) umma_f16(d, q + ((i >> 2) * (QP_ROWS * 128) + 32 * (i & 3)) / 16, k + ((i >> 2) * (QP_KEYS * 128) + 32 * (i & 3)) / 16, id_s, i > 0);
                umma_commit(bar(QP_S, 2 * u + (t & 1)));
            }
        };
        auto values = [&](int t) {
            if (one) {
                const uint64_t v = dv + (t % QP_STAGES) * (2 * L::TILE / 16);
                const uint32_t w = t_unit + 64 * (t & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) umma_f16_ts(t_unit + 128, w + 8 * i, v + 2 * i, id_o, 1);
                umma_commit(bar(QP_O, u));
                umma_commit(bar(QP_FREE, t % QP_STAGES));
            }
        };
        bool ok = wait(bar(QP_QUERY), 0) && wait(bar(QP_FULL, 0), 0);
        if (ok) {
            tc_fence_after();
            scores(0);
        }
        // scores of tile t + 1 go where the weights of tile t - 1 were, once the product that reads those is complete; ahead of the wait for tile t's weights
        for (int t = 0; t < n_tiles && ok; ++t) {
            if (t + 1 < n_tiles) {
                ok = wait(bar(QP_FULL, (t + 1) % QP_STAGES), ((t + 1) / QP_STAGES) & 1);
                if (ok && t > 0) ok = wait(bar(QP_O, u), (t - 1) & 1);
                tc_fence_after();
                if (ok) scores(t + 1);
            }
            ok = ok && wait(bar(QP_P, 2 * u + (t & 1)), (t >> 1) & 1);
            tc_fence_after();
            if (ok) values(t);
        }
        if (!ok) {      // products in flight still read shared and tensor memory
            if (one) umma_commit(bar(QP_DRAIN, u));
            mbar_wait_warp(bar(QP_DRAIN, u), 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) tmem_dealloc(tmem, 512);
}

// The parts of rows whose keys were split, added up: a warp per row of a tile, in the order of the parts.
template <int HD>
__global__ void __launch_bounds__(256) k_q4_join(const PromptParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, G = p.heads / p.n_kv, kvh = blockIdx.y, r = blockIdx.z * 8 + (threadIdx.x >> 5);
    const dc_q4_tile tl = p.tiles[p.joins[blockIdx.x]];
    if (r >= tl.count * G - tl.row0) return;
    constexpr size_t ROW = HD + 4, PART = 2 * QP_ROWS * ROW;
    const float* from = p.ws + ((size_t)tl.ws * p.n_kv + (size_t)tl.n_splits * kvh) * PART + r * ROW;
    constexpr int PER = HD / 32;
    float M = -1e30f, l = 0.0f, v[PER] = {};
    for (int s0 = 0; s0 < tl.n_splits; s0 += 4) {      // four parts' numbers on their way at once
        float2 ml[4];
        float x[4][PER];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float* at = from + (size_t)min(s0 + k, tl.n_splits - 1) * PART;
            ml[k] = __ldcg(reinterpret_cast<const float2*>(at + HD));
            if constexpr (PER == 4) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(at) + lane);
                x[k][0] = f.x, x[k][1] = f.y, x[k][2] = f.z, x[k][3] = f.w;
            } else {
                const float2 f = __ldcg(reinterpret_cast<const float2*>(at) + lane);
                x[k][0] = f.x, x[k][1] = f.y;
            }
        }
        float m = M;
#pragma unroll
        for (int k = 0; k < 4; ++k) m = fmaxf(m, ml[k].x);
        const float old = ex2(M - m);
        M = m, l *= old;
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] *= old;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (s0 + k >= tl.n_splits) break;
            const float f = ex2(ml[k].x - M);
            l = fmaf(ml[k].y, f, l);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = fmaf(x[k][i], f, v[i]);
        }
    }
    const float inv = 1.0f / l;
    const int x = tl.row0 + r, j = x / G;
    __nv_bfloat16* dst = p.out + (size_t)(tl.tok0 + j) * p.ldo + (size_t)(kvh * G + x - j * G) * HD + PER * lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) dst[i] = __float2bfloat16_rn(v[i] * inv);
}

PromptParams params(const dc_q4_call& c) {
    const dc_q4& z = *c.kv->q4;
    return {(const dc_q4_tile*)(z.plan + z.at[DC_Q4_TILES]), (const int32_t*)(z.plan + z.at[DC_Q4_JOINS]), (float*)(z.plan + z.at[DC_Q4_PARTS]),
            (const __nv_bfloat16*)c.q, c.ldq, c.ldo, z.heads, z.kv, c.kv->max_blocks_per_seq, c.kv->d_tables, c.arena, c.scale, (__nv_bfloat16*)c.out};
}

template <int HD>
int launch(dc_ctx* ctx, const dc_q4_call& c) {
    DC_TRY(dc_kernel_setup_unspilled(ctx, (const void*)k_q4_prompt<HD>, (int)Lay<HD>::SMEM, "k_q4_prompt"));
    return dc_launch(ctx, "k_q4_prompt", k_q4_prompt<HD>, dim3(c.kv->q4->kv * c.kv->q4->n_tiles), dim3(QP_THREADS), Lay<HD>::SMEM, params(c), ctx->d_err);
}

}  // namespace

int dc_launch_q4_prompt(dc_ctx* ctx, const dc_q4_call& c) {
    if (c.kv->q4->n_tiles == 0) return DC_B200_OK;
    return c.kv->q4->dim == 128 ? launch<128>(ctx, c) : launch<64>(ctx, c);
}

int dc_launch_q4_join(dc_ctx* ctx, const dc_q4_call& c) {
    const dc_q4& z = *c.kv->q4;
    if (z.n_joins == 0) return DC_B200_OK;
    const dim3 grid(z.n_joins, z.kv, 2 * QP_ROWS / 8);
    return z.dim == 128 ? dc_launch(ctx, "k_q4_join", k_q4_join<128>, grid, dim3(256), 0, params(c)) : dc_launch(ctx, "k_q4_join", k_q4_join<64>, grid, dim3(256), 0, params(c));
}
