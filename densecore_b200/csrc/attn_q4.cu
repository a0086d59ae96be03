// Attention over a paged cache that holds keys and values in 4 bits.
//
// A cached row of a head is held in groups of 64 values: m = fp16(least), d = fp16((largest - least) * fp32(1/15)), codes
// q = rint((x - m) / d) within 0..15 (0 where d is 0), all in fp32; a code stands for fp32(d q + m).  A group with a value that is not
// finite or beyond +-32768 (above it d c + m may leave fp16's range) is held with d = m = NaN, and reads back so.  Blocks, tables, sharing and copy-on-write are kv.cu's, on planes of
// one record per (page, key head) (dc_q4.h).  A step is planned once (dc_b200_kv_batch) and then run for every layer.
//
// Scores of a token: sum over groups of d (q . codes) + m (sum of q); answers: sum over tokens of (p d) codes, plus the sum of p m.  Codes go to the
// tensor cores as fp16, the scales are applied to f32 sums and weights.
//   bf16 rows: codes as they lie (fp16 subnormals c 2^-24 and c 2^-20, exact), queries as fp16 (exact: 8 bits), weights p d rounded to fp16 (half a step, 2^-11 relative,
//   an eighth of a bf16 result's own).  Answers are made transposed, 16 dimensions x 8 rows, which fills the operand's sixteen rows with one word of codes a lane.
// The running reference of a row's exponentials is the largest of score + log2 d (d of the token's value, at least 2^-24), not of the scores: the weights p d stay
// within 64 whatever the values' size, and clear of fp16's least numbers.
//   f32 rows: queries and weights as two fp16 terms (22 bits), rows h and h + 8 of one sixteen-row operand, so that they cost no extra product; codes as c - 8
//   with m + 8 d in place of m: sums around zero, where c and m alone would leave answers as small differences of large sums (measured: 5e-5 of the result, now below 1e-6).
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_launch.cuh"
#include "dc_q4.h"

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
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float2 pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 pair(const __nv_bfloat16* p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p)); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight codes of a word as four pairs: nibbles (0, 4) and (2, 6) times 1, (1, 5) and (3, 7) times 16; EXACT: c - 8, else c 2^-24.
template <bool EXACT>
__device__ __forceinline__ void codes_of(uint32_t w, uint32_t (&c)[4]) {
    const uint32_t w8 = w >> 8;
    if constexpr (EXACT) {
        const __half2 lo = __floats2half2_rn(-1032.0f, -1032.0f), hi = __floats2half2_rn(-1152.0f, -1152.0f);
        auto add = [](uint32_t x, __half2 y) {
            const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&x), y);
            return *reinterpret_cast<const uint32_t*>(&r);
        };
        c[0] = add((w & 0x000F000Fu) | 0x64006400u, lo), c[1] = add((w & 0x00F000F0u) | 0x64006400u, hi);
        c[2] = add((w8 & 0x000F000Fu) | 0x64006400u, lo), c[3] = add((w8 & 0x00F000F0u) | 0x64006400u, hi);
    } else {
        c[0] = w & 0x000F000Fu, c[1] = w & 0x00F000F0u, c[2] = w8 & 0x000F000Fu, c[3] = w8 & 0x00F000F0u;
    }
}

// ---------------------------------------------------------------- new rows into the cache
struct WriteParams {
    const dc_q4_head* head;
    const dc_q4_token* tokens;   // null: the header's
    const void *k, *v;
    int ldkv, n_kv;
    uint8_t* arena;
    float *k_held, *v_held;      // [T][n_kv][HD], may be null
    int few;                     // ahead of captured attention, which does not serve steps with prompt-sized entries: their rows may be more than its buffers hold
};

// rint(x / d) as the division rounds it, x within 16 d: by the reciprocal, and by the division itself where the product lies near a border
__device__ __forceinline__ float rounded_quotient(float x, float d, float inv) {
    const float t = x * inv, q = rintf(t);
    return fabsf(fabsf(t - q) - 0.5f) < 1e-4f ? rintf(__fdiv_rn(x, d)) : q;
}

// One warp per (token, key head), its key and value side by side.  Bound: latency (a step's rows are some KB, about 2 us); a prompt's by its rows.
template <int HD, typename TX>
__global__ void __launch_bounds__(128) k_q4_write(const WriteParams p) {
    using R = dc_q4_rec<HD>;
    constexpr int PER = HD / 32, LANES = 64 / PER;      // neighbouring values of a lane, lanes of a group
    __shared__ uint8_t codes[4][2][HD];
    pdl_wait();
    pdl_launch_dependents();      // (not before the wait: what the next kernel reads ahead of its own wait has to be complete)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, units = p.few && p.head->n_tiles > 0 ? 0 : p.head->T * p.n_kv;
    const dc_q4_token* tokens = p.tokens ? p.tokens : p.head->tokens;
    for (int u = blockIdx.x * 4 + warp; u < units; u += gridDim.x * 4) {
        const int t = u / p.n_kv, head = u - t * p.n_kv;
        const dc_q4_token tok = tokens[t];
        float x[2][PER], lo[2], hi[2];
        bool fine[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const TX* src = reinterpret_cast<const TX*>(w ? p.v : p.k) + (size_t)t * p.ldkv + head * HD + PER * lane;
#pragma unroll
            for (int i = 0; i < PER; ++i) x[w][i] = to_f32(src[i]);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            lo[w] = INFINITY, hi[w] = -INFINITY, fine[w] = true;
#pragma unroll
            for (int i = 0; i < PER; ++i) fine[w] = fine[w] && fabsf(x[w][i]) <= 32768.0f, lo[w] = fminf(lo[w], x[w][i]), hi[w] = fmaxf(hi[w], x[w][i]);
        }
#pragma unroll
        for (int s = LANES / 2; s > 0; s >>= 1)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                lo[w] = fminf(lo[w], __shfl_xor_sync(0xffffffffu, lo[w], s));
                hi[w] = fmaxf(hi[w], __shfl_xor_sync(0xffffffffu, hi[w], s));
            }
        uint8_t* rec = p.arena + ((size_t)tok.block * p.n_kv + head) * R::BYTES;
        __syncwarp();
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t bad = __ballot_sync(0xffffffffu, !fine[w]) >> (lane / LANES * LANES);
            const bool nan = (LANES == 32 ? bad : bad & ((1u << (LANES & 31)) - 1u)) != 0;
            __half d = __float2half_rn(__fmul_rn(__fsub_rn(hi[w], lo[w]), 1.0f / 15.0f)), m = __float2half_rn(lo[w]);
            const float df = __half2float(d), mf = __half2float(m), inv = __fdividef(1.0f, df);
            const bool steps = !nan && df > 0.0f;
            if (nan) d = m = __ushort_as_half((unsigned short)0x7FFF);
            const float ds = __half2float(d), ms = __half2float(m);
            float* held = w ? p.v_held : p.k_held;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float q = steps ? fminf(fmaxf(rounded_quotient(__fsub_rn(x[w][i], mf), df, inv), 0.0f), 15.0f) : 0.0f;
                codes[warp][w][PER * lane + i] = (uint8_t)q;
                x[w][i] = fmaf(ds, q, ms);
            }
            if (held) {
                float* to = held + ((size_t)t * p.n_kv + head) * HD + PER * lane;
#pragma unroll
                for (int i = 0; i < PER; ++i) to[i] = x[w][i];
            }
            if (lane % LANES == 0) reinterpret_cast<__half2*>(rec + (w ? R::V_SCALES : R::K_SCALES))[tok.slot * R::GROUPS + lane / LANES] = __halves2half2(d, m);
        }
        __syncwarp();
        if (lane < HD / 8) {
            const uint8_t* c = codes[warp][0];
            const int t4 = lane & 3, i = lane >> 2;
            uint32_t word = 0;
#pragma unroll
            for (int n = 0; n < 8; ++n) word |= (uint32_t)c[32 * i + 8 * (n & 3) + 2 * t4 + (n >> 2)] << (4 * n);
            *reinterpret_cast<uint32_t*>(rec + R::k_word(tok.slot, t4, i)) = word;
        }
        const uint8_t* c = codes[warp][1];
#pragma unroll
        for (int b = lane; b < HD / 2; b += 32) {
            const int d8 = b & 7, i = b >> 3;
            rec[R::v_byte(tok.slot, d8, i)] = c[16 * i + d8] | (uint8_t)(c[16 * i + 8 + d8] << 4);
        }
    }
}

// ---------------------------------------------------------------- attention, eight rows at a time
struct RowsParams {
    const dc_q4_head* head;
    const dc_q4_item* items;      // these three: not of captured calls
    int* tickets;
    float* ws;
    const void* q;
    int ldq, ldo, heads, n_kv, max_blocks;
    const int32_t* tables;
    const uint8_t* arena;
    float scale;
    void* out;
    int early;      // dc_q4_call
    int* err;
};

constexpr int RW = DC_Q4_WARPS;
constexpr int RW_STAGES = 3;      // pages in flight, per warp
template <int HD>
constexpr size_t rows_smem() { return (size_t)RW * RW_STAGES * dc_q4_rec<HD>::BYTES + RW * RW_STAGES * 8 + (size_t)RW * 8 * (HD + 2) * 4 + HD / 16 * 512; }

// One CTA per (item, key head): its warps take the item's pages in turn, each with a running maximum of its own, and join at the end; the last CTA of a tile joins
// the tile's splits in their order, so that results do not depend on who comes last.
// Bound: a step of few tokens by its launches (one request of 512 positions 10.4 us, sixteen of up to 2300 14.5 us, with the rows' writing; captured ones the same within
// 0.2 us); a long cache by the chain of a page (codes and scales into operands, scores, weights, answers) in 16 warps an SM, f32 12: 48 requests of up to 32000 positions, 533 MB, bf16
// 161 us, 3.3 TB/s, 59 % of the issue slots, half of each score product's sixteen rows empty; f32 211 us.  Four CTAs an SM hold bf16 rows of heads of 128 to 128 registers, of
// which 32 bytes spill.  Four warps a CTA beat eight (sixteen requests 15 against 23 us): fewer parts to join.
// f32 prompts run here too, eight rows at a time, each tile of rows through all pages that it sees: 2011 tokens, 32 query heads, 4 key heads 452 us where k_q4_prompt takes 59
// on bf16 rows (its operands are fp16: f32 rows would need two terms of each).
// A lane has row h = lane / 4 of the tile and tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of a page (t = lane % 4).
// CAPTURED: the arrays' places come from the header, and there may be more CTAs than items.  A step with prompt-sized entries, which it does not serve, is reported.
template <int HD, typename TX, bool CAPTURED>
__global__ void __launch_bounds__(RW * 32, sizeof(TX) == 2 ? 4 : 3) k_q4_rows(const RowsParams p) {
    using R = dc_q4_rec<HD>;
    constexpr bool EXACT = sizeof(TX) == 4;
    constexpr int GR = R::GROUPS, KW = HD / 32, VW = HD / 16, OT = EXACT ? HD / 8 : HD / 16, PART = 8 * (HD + 2);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = lane >> 2, t4 = lane & 3, kvh = blockIdx.y, G = p.heads / p.n_kv;
    const uint32_t ring = smem_u32(smem) + warp * RW_STAGES * R::BYTES, bars = smem_u32(smem) + RW * RW_STAGES * R::BYTES + warp * RW_STAGES * 8;
    float* part = reinterpret_cast<float*>(smem + RW * RW_STAGES * R::BYTES + RW * RW_STAGES * 8);      // [RW][8][HD], then maxima and sums
    float* part_ml = part + RW * 8 * HD;
    // the queries as operands, [16 dimensions][lane]: they would take HD / 8 or HD / 4 registers of every warp
    constexpr int QB = EXACT ? 16 : 8;
    const uint32_t sq = smem_u32(part_ml + RW * 16) + lane * QB;
    if (lane == 0) {
        for (int s = 0; s < RW_STAGES; ++s) mbar_init(bars + 8 * s, 1);
        mbar_fence_init();
    }
    __syncwarp();
    bool waited = !p.early;
    if (waited) pdl_wait();
    pdl_launch_dependents();
    dc_q4_item im;
    if constexpr (!CAPTURED) im = p.items[blockIdx.x];      // (as many as CTAs: it need not wait for their number)
    int n_items = p.head->n_items;
    if (CAPTURED && p.head->n_tiles > 0) {
        n_items = 0;
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicExch(p.err, DC_ERR_REPLAY);
    }
    uint32_t n_full = 0;      // pages that this warp has waited for
    for (int it = blockIdx.x; it < n_items; it += gridDim.x) {
        if (CAPTURED || it != (int)blockIdx.x) im = (CAPTURED ? p.head->items : p.items)[it];
        const int r = im.tile * 8 + h, j = r / G, g = r - j * G;
        const bool row = j < im.count;
        const int qpos = im.pos0 + j, first_new = im.pos0 / DC_KV_BLOCK, all_see = im.pos0 + im.tile * 8 / G;      // positions up to all_see: seen by every row
        const int n_my = (im.page1 - im.page0 - warp + RW - 1) / RW;
        const int32_t* table = p.tables + (size_t)im.seq * p.max_blocks;
        int entry = 0;      // lane i: the block of page (i + a multiple of 32) of this warp
        auto issue = [&](int i) {
            const int page = im.page0 + warp + i * RW;
            if (i % 32 == 0) entry = i + lane < n_my ? table[page + lane * RW] : 0;
            if (!waited && p.early == 1 && page >= first_new) pdl_wait(), waited = true;
            const int block = __shfl_sync(0xffffffffu, entry, i % 32);
            if (lane == 0) {
                const uint32_t s = (n_full + i) % RW_STAGES;
                mbar_expect_tx(bars + 8 * s, R::BYTES);
                bulk_g2s(ring + s * R::BYTES, p.arena + ((size_t)block * p.n_kv + kvh) * R::BYTES, R::BYTES, bars + 8 * s);
            }
        };
#pragma unroll
        for (int i = 0; i < RW_STAGES; ++i)
            if (i < n_my) issue(i);
        // ---- queries as fp16 terms of q 2^(10 - e), 2^e <= largest of the row < 2^(e + 1); dimensions that meet codes times 16 are divided by 16.
        // F turns the products' sums into scores in units of log2 e; qsum: sums of a group's queries in these units
        float qsum[GR], F;
        {
            float x[HD / 16][4], most = 0.0f;
            const TX* src = reinterpret_cast<const TX*>(p.q) + (size_t)(im.tok0 + (row ? j : 0)) * p.ldq + (size_t)(kvh * G + (row ? g : 0)) * HD + 2 * t4;
            const float mul = p.scale * 1.4426950408889634f;
            if (((uintptr_t)src & (2 * sizeof(TX) - 1)) == 0) {
#pragma unroll
                for (int s = 0; s < HD / 8; ++s) {
                    const float2 f = row ? pair(src + 8 * s) : make_float2(0.0f, 0.0f);
                    x[s / 2][2 * (s & 1)] = f.x, x[s / 2][2 * (s & 1) + 1] = f.y;
                }
            } else {
#pragma unroll
                for (int s = 0; s < HD / 16; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[s][i] = row ? to_f32(src[16 * s + 8 * (i >> 1) + (i & 1)]) : 0.0f;
            }
#pragma unroll
            for (int s = 0; s < GR; ++s) qsum[s] = 0.0f;
#pragma unroll
            for (int s = 0; s < HD / 16; ++s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    most = fmaxf(most, fabsf(x[s][i]));
                    qsum[s / 4] += x[s][i];
                }
            }
#pragma unroll
            for (int s = 1; s < 4; s <<= 1) {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
#pragma unroll
                for (int i = 0; i < GR; ++i) qsum[i] += __shfl_xor_sync(0xffffffffu, qsum[i], s);
            }
#pragma unroll
            for (int i = 0; i < GR; ++i) qsum[i] *= mul;
            const int e = max(-100, min(100, (int)(__float_as_uint(most) >> 23) - 127));
            const float up = __uint_as_float((uint32_t)(137 - e) << 23);
            F = __uint_as_float((uint32_t)((EXACT ? 117 : 141) + e) << 23) * mul;
#pragma unroll
            for (int s = 0; s < HD / 16; ++s) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = x[s][2 * i] * (i ? up * 0.0625f : up), b = x[s][2 * i + 1] * (i ? up * 0.0625f : up);
                    w[2 * i] = pack_h2(a, b);
                    if constexpr (EXACT) {
                        const float2 f = unpack_h2(w[2 * i]);
                        w[2 * i + 1] = pack_h2(a - f.x, b - f.y);
                    }
                }
                if (warp == s % RW) {
                    if constexpr (EXACT) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sq + 32 * QB * s), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                    else asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(sq + 32 * QB * s), "r"(w[0]), "r"(w[2]) : "memory");
                }
            }
            __syncthreads();
        }
        // EXACT: tile c of o has dimensions 8 c + 2 t, + 1 of rows h (first terms) and h (second terms); else dimensions 16 c + h and + 8 of rows 2 t, + 1
        float o[OT][4], om[GR], m_run = -1e30f, l = 0.0f;
#pragma unroll
        for (int i = 0; i < OT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < GR; ++i) om[i] = 0.0f;

        for (int i = 0; i < n_my; ++i) {
            const uint32_t s = (n_full + i) % RW_STAGES, at = ring + s * R::BYTES;
            mbar_wait(bars + 8 * s, ((n_full + i) / RW_STAGES) & 1, p.err);
            // ---- the page into registers, its stage to the next one
            uint32_t kw[2][KW], vw[VW], kd[2][2][GR], vd[2][2][GR];      // [half][token of two]
            if constexpr (HD == 128) {
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const uint4 x = lds128(at + a * 512 + lane * 16), y = lds128(at + R::V_CODES + a * 512 + lane * 16);
                    kw[a][0] = x.x, kw[a][1] = x.y, kw[a][2] = x.z, kw[a][3] = x.w;
                    vw[4 * a] = y.x, vw[4 * a + 1] = y.y, vw[4 * a + 2] = y.z, vw[4 * a + 3] = y.w;
                    const uint4 u = lds128(at + R::K_SCALES + (8 * a + 2 * t4) * 8), w = lds128(at + R::V_SCALES + (8 * a + 2 * t4) * 8);
                    kd[a][0][0] = u.x, kd[a][0][1] = u.y, kd[a][1][0] = u.z, kd[a][1][1] = u.w;
                    vd[a][0][0] = w.x, vd[a][0][1] = w.y, vd[a][1][0] = w.z, vd[a][1][1] = w.w;
                }
            } else {
                const uint4 x = lds128(at + lane * 16), y = lds128(at + R::V_CODES + lane * 16);
                kw[0][0] = x.x, kw[0][1] = x.y, kw[1][0] = x.z, kw[1][1] = x.w;
                vw[0] = y.x, vw[1] = y.y, vw[2] = y.z, vw[3] = y.w;
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const uint2 u = lds64(at + R::K_SCALES + (8 * a + 2 * t4) * 4), w = lds64(at + R::V_SCALES + (8 * a + 2 * t4) * 4);
                    kd[a][0][0] = u.x, kd[a][1][0] = u.y, vd[a][0][0] = w.x, vd[a][1][0] = w.y;
                }
            }
            __syncwarp();
            if (i + RW_STAGES < n_my) issue(i + RW_STAGES);
            // ---- scores
            float sc[2][2], mx = -INFINITY;
            const int pos = (im.page0 + warp + i * RW) * DC_KV_BLOCK;
            float acc[2][GR][4];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int c = 0; c < GR; ++c) acc[a][c][0] = acc[a][c][1] = acc[a][c][2] = acc[a][c][3] = 0.0f;
            // (groups and halves in turn: a product does not wait for the one before)
#pragma unroll
            for (int k = 0; k < KW / GR; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int g = 0; g < GR; ++g) {
                        const int c = g * (KW / GR) + k;
                        uint32_t q4[4];
                        if constexpr (EXACT) {
                            const uint4 f = lds128(sq + 32 * QB * (2 * c + half));
                            q4[0] = f.x, q4[1] = f.y, q4[2] = f.z, q4[3] = f.w;
                        } else {
                            const uint2 f = lds64(sq + 32 * QB * (2 * c + half));
                            q4[0] = f.x, q4[1] = 0u, q4[2] = f.y, q4[3] = 0u;
                        }
#pragma unroll
                        for (int a = 0; a < 2; ++a) {
                            uint32_t b[4];
                            codes_of<EXACT>(kw[a][c], b);
                            mma_f16(acc[a][g], q4, b[2 * half], b[2 * half + 1]);
                        }
                    }
#pragma unroll
            for (int a = 0; a < 2; ++a) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float x = 0.0f, y = 0.0f;
#pragma unroll
                    for (int c = 0; c < GR; ++c) {
                        const float2 dm = unpack_h2(kd[a][b][c]);
                        x = fmaf(dm.x, EXACT ? acc[a][c][b] + acc[a][c][2 + b] : acc[a][c][b], x);
                        y = fmaf(EXACT ? fmaf(8.0f, dm.x, dm.y) : dm.y, qsum[c], y);
                    }
                    sc[a][b] = fmaf(x, F, y);
                }
            }
            if (pos + DC_KV_BLOCK - 1 > all_see) {      // some row does not see all of the page; what lies there may be anything
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        if (pos + 8 * a + 2 * t4 + b > qpos) {
                            sc[a][b] = -INFINITY;
#pragma unroll
                            for (int c = 0; c < GR; ++c) vd[a][b][c] = 0;
                        }
            }
            float2 dm[2][2][GR];      // values' scales and least ones (EXACT: the middle, m + 8 d)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float most = 0.0f;
#pragma unroll
                    for (int c = 0; c < GR; ++c) {
                        dm[a][b][c] = unpack_h2(vd[a][b][c]);
                        if constexpr (EXACT) dm[a][b][c].y = fmaf(8.0f, dm[a][b][c].x, dm[a][b][c].y);
                        most = fmaxf(most, dm[a][b][c].x);
                    }
                    mx = fmaxf(mx, sc[a][b] + fmaxf(lg2(most), -24.0f));
                }
            // (the reference follows once it is 2^6 behind: weights up to 64 are as exact, and the row's maximum and the answers' factors are rare)
            if (__any_sync(0xffffffffu, mx > m_run + 6.0f)) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float m_new = fmaxf(m_run, mx), corr = ex2(m_run - m_new);
                m_run = m_new;
                l *= corr;
#pragma unroll
                for (int c = 0; c < GR; ++c) om[c] *= corr;
                if constexpr (EXACT) {
#pragma unroll
                    for (int c = 0; c < OT; ++c) o[c][0] *= corr, o[c][1] *= corr, o[c][2] *= corr, o[c][3] *= corr;
                } else {
                    const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t4), c1 = __shfl_sync(0xffffffffu, corr, 8 * t4 + 4);
#pragma unroll
                    for (int c = 0; c < OT; ++c) o[c][0] *= c0, o[c][1] *= c1, o[c][2] *= c0, o[c][3] *= c1;
                }
            }
            // ---- weights times scales, values
            uint32_t pa[GR][EXACT ? 4 : 2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const float p0 = ex2(sc[a][0] - m_run), p1 = ex2(sc[a][1] - m_run);
                l += p0 + p1;
#pragma unroll
                for (int c = 0; c < GR; ++c) {
                    const float2 d0 = dm[a][0][c], d1 = dm[a][1][c];
                    om[c] = fmaf(p0, d0.y, om[c]);
                    om[c] = fmaf(p1, d1.y, om[c]);
                    const float w0 = p0 * d0.x, w1 = p1 * d1.x;
                    const uint32_t hi = pack_h2(w0, w1);
                    if constexpr (EXACT) {      // the second term 2^11 fold: it stays clear of fp16's least numbers
                        const float2 f = unpack_h2(hi);
                        pa[c][2 * a] = hi;
                        pa[c][2 * a + 1] = pack_h2((w0 - f.x) * 2048.0f, (w1 - f.y) * 2048.0f);
                    } else {
                        pa[c][a] = hi;
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < VW; ++c) {
                uint32_t b[4];
                codes_of<EXACT>(vw[c], b);
                if constexpr (EXACT) {
                    mma_f16(o[2 * c], pa[c / 4], b[0], b[2]);
                    mma_f16(o[2 * c + 1], pa[c / 4], b[1], b[3]);
                } else {
                    mma_f16(o[c], b, pa[c / 4][0], pa[c / 4][1]);
                }
            }
        }
        n_full += max(0, n_my);
        // ---- the warps' parts
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, s);
#pragma unroll
            for (int c = 0; c < GR; ++c) om[c] += __shfl_xor_sync(0xffffffffu, om[c], s);
        }
        if constexpr (EXACT) {
#pragma unroll
            for (int c = 0; c < OT; ++c) {
                const float f = c & 1 ? 0.0625f : 1.0f;
                float2 x;
                x.x = fmaf(fmaf(o[c][2], 1.0f / 2048.0f, o[c][0]), f, om[c / 8]);
                x.y = fmaf(fmaf(o[c][3], 1.0f / 2048.0f, o[c][1]), f, om[c / 8]);
                *reinterpret_cast<float2*>(part + (warp * 8 + h) * HD + 8 * c + 2 * t4) = x;
            }
        } else {
            float om2[GR][2];
#pragma unroll
            for (int c = 0; c < GR; ++c) om2[c][0] = __shfl_sync(0xffffffffu, om[c], 8 * t4), om2[c][1] = __shfl_sync(0xffffffffu, om[c], 8 * t4 + 4);
#pragma unroll
            for (int c = 0; c < OT; ++c) {
                float* to = part + (warp * 8 + 2 * t4) * HD + 16 * c + h;
                to[0] = fmaf(o[c][0], 16777216.0f, om2[c / 4][0]);
                to[HD] = fmaf(o[c][1], 16777216.0f, om2[c / 4][1]);
                to[8] = fmaf(o[c][2], 1048576.0f, om2[c / 4][0]);
                to[HD + 8] = fmaf(o[c][3], 1048576.0f, om2[c / 4][1]);
            }
        }
        if (t4 == 0) part_ml[2 * (warp * 8 + h)] = m_run, part_ml[2 * (warp * 8 + h) + 1] = l;
        if (!waited && p.early == 1) pdl_wait(), waited = true;      // (ahead of the first store)
        __syncthreads();
        // ---- joined: a thread has four neighbouring dimensions of a row at a time
        const bool alone = im.n_splits == 1;
        float* ws = (CAPTURED ? p.head->ws : p.ws) + ((size_t)im.ws * p.n_kv + (size_t)im.n_splits * kvh) * PART;
        auto store = [&](int x4, const float4& v, float inv) {
            const int ro = im.tile * 8 + x4 / (HD / 4), jo = ro / G, go = ro - jo * G;
            if (jo >= im.count) return;
            TX* to = reinterpret_cast<TX*>(p.out) + (size_t)(im.tok0 + jo) * p.ldo + (size_t)(kvh * G + go) * HD + 4 * (x4 % (HD / 4));
            put(to, v.x * inv), put(to + 1, v.y * inv), put(to + 2, v.z * inv), put(to + 3, v.w * inv);
        };
        for (int x4 = threadIdx.x; x4 < 8 * HD / 4; x4 += RW * 32) {
            const int rr = x4 / (HD / 4);
            float M = -1e30f, L = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < RW; ++w) M = fmaxf(M, part_ml[2 * (w * 8 + rr)]);
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                const float f = ex2(part_ml[2 * (w * 8 + rr)] - M);
                const float4 x = reinterpret_cast<const float4*>(part + w * 8 * HD)[x4];
                L = fmaf(part_ml[2 * (w * 8 + rr) + 1], f, L);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
            }
            if (alone) {
                store(x4, v, __fdividef(1.0f, L));
            } else {
                float* to = ws + (size_t)im.split * PART;
                reinterpret_cast<float4*>(to)[x4] = v;
                if (x4 % (HD / 4) == 0) to[8 * HD + rr] = M, to[8 * HD + 8 + rr] = L;
            }
        }
        if (!alone) {
            int* ticket = (CAPTURED ? p.head->tickets : p.tickets) + im.ticket * p.n_kv + kvh;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                s_last = atomicAdd(ticket, 1) == im.n_splits - 1;
                if (s_last) *ticket = 0;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                // the splits' factors in place of the parts: [split][8 rows], DC_Q4_SPLITS at most; then rows' sums.  The first splits' sums are on their way meanwhile
                static_assert(DC_Q4_SPLITS * 8 + 8 <= RW * 8 * 64 && 8 * HD / 4 % (RW * 32) == 0, "factors take the parts' place");
                constexpr int AHEAD = 2, X4 = 8 * HD / 4 / (RW * 32);
                float4 first[X4][AHEAD];
#pragma unroll
                for (int k = 0; k < X4; ++k)
#pragma unroll
                    for (int s = 0; s < AHEAD; ++s)
                        if (s < im.n_splits) first[k][s] = __ldcg(reinterpret_cast<const float4*>(ws + (size_t)s * PART) + threadIdx.x + k * RW * 32);
                float *f = part, *inv = part + DC_Q4_SPLITS * 8;
                if (threadIdx.x < 32) {
                    const int rr = lane & 7;      // four lanes a row
                    float M = -1e30f, L = 0.0f;
                    const float m0 = lane >> 3 < im.n_splits ? __ldcg(ws + (size_t)(lane >> 3) * PART + 8 * HD + rr) : -1e30f;
                    const float l0 = lane >> 3 < im.n_splits ? __ldcg(ws + (size_t)(lane >> 3) * PART + 8 * HD + 8 + rr) : 0.0f;
                    M = m0;
                    for (int s = (lane >> 3) + 4; s < im.n_splits; s += 4) M = fmaxf(M, f[8 * s + rr] = __ldcg(ws + (size_t)s * PART + 8 * HD + rr));
                    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 8));
                    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
                    if (lane >> 3 < im.n_splits) L = l0 * (f[lane] = ex2(m0 - M));
                    for (int s = (lane >> 3) + 4; s < im.n_splits; s += 4) {
                        const float x = ex2(f[8 * s + rr] - M);
                        f[8 * s + rr] = x;
                        L = fmaf(__ldcg(ws + (size_t)s * PART + 8 * HD + 8 + rr), x, L);
                    }
                    L += __shfl_xor_sync(0xffffffffu, L, 8);
                    L += __shfl_xor_sync(0xffffffffu, L, 16);
                    if (lane < 8) inv[rr] = __fdividef(1.0f, L);
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < X4; ++k) {
                    const int x4 = threadIdx.x + k * RW * 32, rr4 = x4 / (HD / 4);
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int s = 0; s < AHEAD; ++s)
                        if (s < im.n_splits) {
                            const float w = f[8 * s + rr4];
                            v.x = fmaf(first[k][s].x, w, v.x), v.y = fmaf(first[k][s].y, w, v.y), v.z = fmaf(first[k][s].z, w, v.z), v.w = fmaf(first[k][s].w, w, v.w);
                        }
#pragma unroll 4
                    for (int s = AHEAD; s < im.n_splits; ++s) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(ws + (size_t)s * PART) + x4);
                        const float w = f[8 * s + rr4];
                        v.x = fmaf(x.x, w, v.x), v.y = fmaf(x.y, w, v.y), v.z = fmaf(x.z, w, v.z), v.w = fmaf(x.w, w, v.w);
                    }
                    store(x4, v, inv[rr4]);
                }
            }
        }
        __syncthreads();      // the parts are free for the next item
    }
    if (!waited) pdl_wait();      // (a successor that waits for this kernel waits for its predecessor too)
}

template <int HD, typename TX>
int launch_rows(dc_ctx* ctx, const dc_q4_call& c) {
    const dc_q4& z = *c.kv->q4;
    const auto kernel = c.captured ? k_q4_rows<HD, TX, true> : k_q4_rows<HD, TX, false>;
    DC_TRY(dc_kernel_setup(ctx, (const void*)kernel, (int)rows_smem<HD>(), "k_q4_rows"));
    const RowsParams p = {z.head, (const dc_q4_item*)(z.plan + z.at[DC_Q4_ITEMS]), (int*)(z.plan + z.at[DC_Q4_TICKETS]), (float*)(z.plan + z.at[DC_Q4_WS]), c.q, c.ldq, c.ldo, z.heads, z.kv, c.kv->max_blocks_per_seq, c.kv->d_tables, c.arena, c.scale, c.out, c.early, ctx->d_err};
    // (a captured call's later plans may have more items: CTAs for all SMs)
    const int ctas = c.captured ? std::max(z.n_items, ((sizeof(TX) == 2 ? 4 : 3) * ctx->num_sms + z.kv - 1) / z.kv) : z.n_items;
    return dc_launch(ctx, "k_q4_rows", kernel, dim3(ctas, z.kv), dim3(RW * 32), rows_smem<HD>(), p);
}

template <int HD, typename TX>
int launch_write(dc_ctx* ctx, const WriteParams& p, int units) {
    return dc_launch(ctx, "k_q4_write", k_q4_write<HD, TX>, dim3(std::min((units + 3) / 4, ctx->num_sms * 8)), dim3(128), 0, p);
}

}  // namespace

int dc_launch_q4_rows(dc_ctx* ctx, const dc_q4_call& c) {
    const dc_q4& z = *c.kv->q4;
    if (z.n_items == 0) return DC_B200_OK;
    if (z.dim == 128) return z.type == DC_TYPE_F32 ? launch_rows<128, float>(ctx, c) : launch_rows<128, __nv_bfloat16>(ctx, c);
    return z.type == DC_TYPE_F32 ? launch_rows<64, float>(ctx, c) : launch_rows<64, __nv_bfloat16>(ctx, c);
}

// ---------------------------------------------------------------- plans
void dc_q4_release(dc_kv_cache* kv) {
    dc_q4* z = kv->q4;
    if (!z) return;
    if (z->plan) cudaFree(z->plan);
    for (uint8_t* p : z->retired) cudaFree(p);
    if (z->head) cudaFree(z->head);
    if (z->stage) cudaFreeHost(z->stage);
    if (z->uploaded) cudaEventDestroy(z->uploaded);
    delete z;
    kv->q4 = nullptr;
}

namespace {

bool capturing(dc_ctx* ctx) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(ctx->stream, &st) == cudaSuccess && st != cudaStreamCaptureStatusNone;
}

// Blocks that the entries need beside the ones they hold: new ones, and copies of the ones they are about to write that someone else holds too.
int blocks_needed(const dc_kv_cache* kv, const std::vector<dc_q4_entry>& es) {
    std::vector<std::pair<int, int>> given;      // (block, references already given up)
    int n = 0;
    for (const dc_q4_entry& e : es) {
        const dc_kv_seq& s = kv->seqs[e.seq];
        const int need = (e.pos0 + e.count + DC_KV_BLOCK - 1) / DC_KV_BLOCK, have = (int)s.blocks.size();
        for (int b = e.pos0 / DC_KV_BLOCK; b < need && b < have; ++b) {
            if (kv->ref[s.blocks[b]] <= 1) continue;
            auto it = std::find_if(given.begin(), given.end(), [&](const std::pair<int, int>& x) { return x.first == s.blocks[b]; });
            if (it == given.end()) it = given.insert(given.end(), {s.blocks[b], 0});
            if (kv->ref[s.blocks[b]] - it->second <= 1) continue;
            ++it->second;
            ++n;
        }
        n += std::max(0, need - have);
    }
    return n;
}

int make_plan(dc_ctx* ctx, dc_kv_cache* kv, const std::vector<dc_q4_entry>& es, int T) {
    dc_q4& z = *kv->q4;
    std::vector<dc_q4_token> tokens(T);
    std::vector<dc_q4_item> items;
    std::vector<dc_q4_tile> tiles;
    std::vector<int32_t> joins;      // tiles whose keys are split: their first part
    const int G = z.heads / z.kv;
    std::vector<dc_q4_entry> few, many;
    for (const dc_q4_entry& e : es) {
        for (int i = 0; i < e.count; ++i) tokens[e.tok0 + i] = {kv->seqs[e.seq].blocks[(e.pos0 + i) / DC_KV_BLOCK], (e.pos0 + i) % DC_KV_BLOCK};
        (z.type == DC_TYPE_BF16 && (long long)e.count * G >= DC_Q4_PROMPT_ROWS ? many : few).push_back(e);
    }
    int n_tickets, n_ws, n_parts;
    dc_q4_items(few, G, z.kv, ctx->num_sms, &items, &n_tickets, &n_ws);
    dc_q4_tiles(many, G, z.kv, ctx->num_sms, &tiles, &n_parts);
    for (size_t i = 0; i < tiles.size(); ++i)
        if (tiles[i].n_splits > 1 && tiles[i].split == 0) joins.push_back((int32_t)i);
    // ---- arrays, tickets (zero, and left so by every call), partial results
    const size_t need[DC_Q4_ARRAYS] = {tokens.size() * sizeof(dc_q4_token), items.size() * sizeof(dc_q4_item), tiles.size() * sizeof(dc_q4_tile), joins.size() * 4, (size_t)n_tickets * z.kv * 4,
                                       (size_t)n_ws * z.kv * 8 * (z.dim + 2) * 4, (size_t)n_parts * z.kv * 256 * (z.dim + 4) * 4};
    bool fits = z.plan != nullptr;
    for (int i = 0; i < DC_Q4_ARRAYS; ++i) fits = fits && need[i] <= z.cap[i];
    if (!fits) {
        size_t cap[DC_Q4_ARRAYS], at[DC_Q4_ARRAYS], bytes = 0;
        for (int i = 0; i < DC_Q4_ARRAYS; ++i) {
            cap[i] = std::max(z.cap[i], (need[i] + need[i] / 2 + 4096) / 256 * 256);
            at[i] = bytes;
            bytes += cap[i];
        }
        z.retired.reserve(z.retired.size() + 1);
        uint8_t* fresh = nullptr;
        DC_TRY(dc_check_cuda(ctx, cudaMalloc(&fresh, bytes), "kv_batch: plan"));
        const cudaError_t e = cudaMemsetAsync(fresh, 0, at[DC_Q4_WS], ctx->stream);
        if (e != cudaSuccess) {
            cudaFree(fresh);
            return dc_check_cuda(ctx, e, "kv_batch: plan");
        }
        if (z.plan) z.retired.push_back(z.plan);
        z.plan = fresh;
        std::copy(cap, cap + DC_Q4_ARRAYS, z.cap), std::copy(at, at + DC_Q4_ARRAYS, z.at);
    }
    if (!z.uploaded) DC_TRY(dc_check_cuda(ctx, cudaEventCreateWithFlags(&z.uploaded, cudaEventDisableTiming), "kv_batch: event"));
    else DC_TRY(dc_check_cuda(ctx, cudaEventSynchronize(z.uploaded), "kv_batch: staging"));
    const size_t staged = sizeof(dc_q4_head) + need[0] + need[1] + need[2] + need[3];
    if (staged > z.stage_bytes) {
        if (z.stage) cudaFreeHost(z.stage);
        z.stage = nullptr, z.stage_bytes = 0;
        DC_TRY(dc_check_cuda(ctx, cudaMallocHost(&z.stage, staged * 2), "kv_batch: staging"));
        z.stage_bytes = staged * 2;
    }
    const dc_q4_head hd = {T, (int)items.size(), (int)tiles.size(), (int)joins.size(), (const dc_q4_token*)(z.plan + z.at[DC_Q4_TOKENS]), (const dc_q4_item*)(z.plan + z.at[DC_Q4_ITEMS]),
                           (int32_t*)(z.plan + z.at[DC_Q4_TICKETS]), (float*)(z.plan + z.at[DC_Q4_WS])};
    const void* from[4] = {tokens.data(), items.data(), tiles.data(), joins.data()};
    size_t off = sizeof(hd);
    for (int i = 0; i < 4; ++i) {
        if (!need[i]) continue;
        memcpy(z.stage + off, from[i], need[i]);
        DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(z.plan + z.at[i], z.stage + off, need[i], cudaMemcpyHostToDevice, ctx->stream), "kv_batch: plan"));
        off += need[i];
    }
    memcpy(z.stage, &hd, sizeof(hd));
    DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(z.head, z.stage, sizeof(hd), cudaMemcpyHostToDevice, ctx->stream), "kv_batch: plan"));
    DC_TRY(dc_check_cuda(ctx, cudaEventRecord(z.uploaded, ctx->stream), "kv_batch: plan"));
    z.T = T, z.n_items = hd.n_items, z.n_tiles = hd.n_tiles, z.n_joins = hd.n_joins;
    return DC_B200_OK;
}

int check_call(dc_ctx* ctx, const dc_kv_cache* kv, int layer, const char* name) {
    if (!ctx || !kv) return DC_B200_INVALID_ARGUMENT;
    if (!kv->q4) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: not a cache in 4 bits", name);
    if (kv->ctx != ctx) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: the cache belongs to another context", name);
    if (layer < 0 || layer >= kv->q4->n_layer) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: layer %d of %d", name, layer, kv->q4->n_layer);
    if (!kv->q4->planned) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: no batch (dc_b200_kv_batch)", name);
    if (kv->q4->edits != kv->edits)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: a sequence was freed, forked, reserved or looked up in the prefix cache since dc_b200_kv_batch", name);
    return DC_B200_OK;
}

int empty_step(dc_ctx* ctx, const char* name) {      // nothing to do; a capture of it would do nothing for later steps either
    return capturing(ctx) ? dc_fail(ctx, DC_B200_UNSUPPORTED, "%s: a step without tokens cannot be captured", name) : DC_B200_OK;
}

int write_rows(dc_ctx* ctx, dc_kv_cache* kv, int layer, const void* k, const void* v, int ldkv, float* k_held, float* v_held, bool captured, bool few) {
    const dc_q4& z = *kv->q4;
    const WriteParams p = {z.head, captured ? nullptr : (const dc_q4_token*)(z.plan + z.at[DC_Q4_TOKENS]), k, v, ldkv, z.kv, kv->planes[layer].arena, k_held, v_held, few};
    const int units = z.T * z.kv;
    if (z.dim == 128) return z.type == DC_TYPE_F32 ? launch_write<128, float>(ctx, p, units) : launch_write<128, __nv_bfloat16>(ctx, p, units);
    return z.type == DC_TYPE_F32 ? launch_write<64, float>(ctx, p, units) : launch_write<64, __nv_bfloat16>(ctx, p, units);
}

int create(dc_ctx* ctx, dc_kv_cache* kv, int n_layer, int n_head, int n_kv_head, int head_dim, int row_type, int max_blocks, int max_seqs, int max_blocks_per_seq) {
    DC_TRY(dc_check_cuda(ctx, cudaMalloc(&kv->q4->head, sizeof(dc_q4_head)), "kv_create_q4"));
    DC_TRY(dc_check_cuda(ctx, cudaMemsetAsync(kv->q4->head, 0, sizeof(dc_q4_head), ctx->stream), "kv_create_q4"));
    kv->q4->n_layer = n_layer, kv->q4->heads = n_head, kv->q4->kv = n_kv_head, kv->q4->dim = head_dim, kv->q4->type = row_type;
    return dc_kv_init_planes(ctx, kv, std::vector<size_t>(n_layer, (size_t)n_kv_head * 18 * head_dim / DC_KV_BLOCK), 0, max_blocks, max_seqs, max_blocks_per_seq);
}

// dc_b200_kv_batch behind its first checks; throws std::bad_alloc.
int begin_step(dc_ctx* ctx, dc_kv_cache* kv, int n_entries, const int32_t* seqs, const int32_t* pos0, const int32_t* counts) {
    std::vector<dc_q4_entry> es;
    std::vector<char> seen(kv->max_seqs, 0);
    long long T = 0;
    for (int i = 0; i < n_entries; ++i) {
        const int s = seqs[i];
        if (s < 0 || s >= kv->max_seqs || !kv->seqs[s].used) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_batch: sequence %d is not allocated", s);
        if (seen[s]) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_batch: sequence %d is named twice", s);
        seen[s] = 1;
        if (counts[i] < 0 || pos0[i] < 0 || pos0[i] > kv->seqs[s].len)
            return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_batch: sequence %d holds %d tokens, asked are %d from position %d on", s, kv->seqs[s].len, counts[i], pos0[i]);
        if ((long long)pos0[i] + counts[i] > (long long)kv->max_blocks_per_seq * DC_KV_BLOCK)
            return dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "kv_batch: sequence %d needs %lld positions, its table holds %d pages", s, (long long)pos0[i] + counts[i], kv->max_blocks_per_seq);
        if (counts[i]) es.push_back({s, pos0[i], counts[i], (int)T});
        T += counts[i];
        if (T * kv->q4->heads > (1 << 30)) return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_batch: more than 2^30 new rows of queries at once");
    }
    const int need = blocks_needed(kv, es), there = dc_kv_available_blocks(kv);
    if (need > there) return dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "kv_batch: out of blocks (%d free, %d needed)", there, need);
    kv->q4->planned = false;
    struct Lengths {      // as they were, should anything fail from here on (blocks reserved meanwhile stay with their sequences)
        dc_kv_cache* kv;
        std::vector<std::pair<int, int>> of;
        ~Lengths() {
            for (const auto& x : of) kv->seqs[x.first].len = x.second;
        }
    } before = {kv, {}};
    for (const dc_q4_entry& e : es) before.of.push_back({e.seq, kv->seqs[e.seq].len});
    for (const dc_q4_entry& e : es) {
        kv->seqs[e.seq].len = e.pos0;      // rows from there on are written anew (what others share is copied first)
        DC_TRY(dc_kv_seq_reserve(kv, e.seq, e.pos0 + e.count));
        kv->seqs[e.seq].len = e.pos0 + e.count;
    }
    DC_TRY(make_plan(ctx, kv, es, (int)T));
    before.of.clear();
    kv->q4->edits = kv->edits;
    kv->q4->planned = true;
    return DC_B200_OK;
}

}  // namespace

extern "C" {

int dc_b200_kv_create_q4(dc_ctx* ctx, int n_layer, int n_head, int n_kv_head, int head_dim, int row_type, int max_blocks, int max_seqs,
                         int max_blocks_per_seq, dc_kv_cache** out) {
    if (!ctx || !out) return DC_B200_INVALID_ARGUMENT;
    *out = nullptr;
    if (n_layer < 1 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || n_kv_head > 65535 || max_blocks < 1 || max_seqs < 1 || max_blocks_per_seq < 1)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_create_q4: bad shape (%d heads, %d key heads)", n_head, n_kv_head);
    if (head_dim != 64 && head_dim != 128) return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_create_q4: head size %d (64 and 128 are supported)", head_dim);
    if (row_type != DC_TYPE_F32 && row_type != DC_TYPE_BF16) return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_create_q4: row type %d (F32 and BF16 are supported)", row_type);
    if (n_head > (1 << 20) || (long long)max_blocks_per_seq * DC_KV_BLOCK > (1 << 30) || (long long)max_seqs * max_blocks_per_seq > (1LL << 31) - 1)
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_create_q4: %d sequences of %d pages, %d heads", max_seqs, max_blocks_per_seq, n_head);
    cudaSetDevice(ctx->device);
    dc_kv_cache* kv = nullptr;
    int st;
    try {
        kv = new dc_kv_cache();
        kv->q4 = new dc_q4();
        st = create(ctx, kv, n_layer, n_head, n_kv_head, head_dim, row_type, max_blocks, max_seqs, max_blocks_per_seq);
    } catch (const std::bad_alloc&) {
        st = dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "kv_create_q4: out of host memory");
    }
    if (st != DC_B200_OK && kv) {
        dc_kv_release(kv);
        delete kv;
        kv = nullptr;
    }
    *out = kv;
    return st;
}

int dc_b200_kv_batch(dc_kv_cache* kv, int n_entries, const int32_t* seqs, const int32_t* pos0, const int32_t* counts) {
    if (!kv) return DC_B200_INVALID_ARGUMENT;
    dc_ctx* ctx = kv->ctx;
    if (!kv->q4) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_batch: not a cache in 4 bits");
    if (n_entries < 0 || (n_entries && (!seqs || !pos0 || !counts))) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_batch: bad argument (%d entries)", n_entries);
    cudaSetDevice(ctx->device);
    if (capturing(ctx)) return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_batch: not within a stream capture");
    try {
        return begin_step(ctx, kv, n_entries, seqs, pos0, counts);
    } catch (const std::bad_alloc&) {
        return dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "kv_batch: out of host memory");
    }
}

int dc_b200_kv_q4_write_dev(dc_ctx* ctx, dc_kv_cache* kv, int layer, const void* k_dev, const void* v_dev, int ld_kv, float* k_held_dev, float* v_held_dev) {
    DC_TRY(check_call(ctx, kv, layer, "kv_q4_write_dev"));
    const dc_q4& z = *kv->q4;
    if (ld_kv == 0) ld_kv = z.kv * z.dim;
    if (z.T == 0) return empty_step(ctx, "kv_q4_write_dev");
    if (!k_dev || !v_dev || ld_kv < z.kv * z.dim) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_q4_write_dev: bad argument (row stride %d)", ld_kv);
    cudaSetDevice(ctx->device);
    return write_rows(ctx, kv, layer, k_dev, v_dev, ld_kv, k_held_dev, v_held_dev, capturing(ctx), false);
}

int dc_b200_flash_attn_q4_dev(dc_ctx* ctx, dc_kv_cache* kv, int layer, const void* q_dev, int ld_q, const void* k_dev, const void* v_dev, int ld_kv, float scale,
                              void* out_dev, int ld_out, float* k_held_dev, float* v_held_dev) {
    DC_TRY(check_call(ctx, kv, layer, "flash_attn_q4_dev"));
    const dc_q4& z = *kv->q4;
    if (ld_q == 0) ld_q = z.heads * z.dim;
    if (ld_kv == 0) ld_kv = z.kv * z.dim;
    if (ld_out == 0) ld_out = z.heads * z.dim;
    if (z.T == 0) return empty_step(ctx, "flash_attn_q4_dev");
    if (!q_dev || !out_dev || (!k_dev != !v_dev) || ld_q < z.heads * z.dim || ld_out < z.heads * z.dim || ld_kv < z.kv * z.dim || (!k_dev && (k_held_dev || v_held_dev)))
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "flash_attn_q4_dev: bad argument (row strides %d, %d, %d)", ld_q, ld_kv, ld_out);
    const bool captured = capturing(ctx);
    if (z.n_tiles && captured) return dc_fail(ctx, DC_B200_UNSUPPORTED, "flash_attn_q4_dev: prompt-sized portions cannot be captured (their number of CTAs goes by the positions)");
    if (!isfinite(scale)) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "flash_attn_q4_dev: scale is not finite");
    cudaSetDevice(ctx->device);
    if (k_dev) DC_TRY(write_rows(ctx, kv, layer, k_dev, v_dev, ld_kv, k_held_dev, v_held_dev, captured, captured));
    dc_q4_call c = {kv, kv->planes[layer].arena, q_dev, ld_q, ld_out, scale, out_dev, k_dev ? 1 : 0, captured};
    DC_TRY(dc_launch_q4_prompt(ctx, c));
    if (z.n_tiles) c.early = 2;      // the SMs that prompt tiles leave idle take the single tokens meanwhile
    DC_TRY(dc_launch_q4_rows(ctx, c));
    return dc_launch_q4_join(ctx, c);
}

int dc_b200_flash_attn_q4(dc_ctx* ctx, dc_kv_cache* kv, int layer, const void* q_host, const void* k_host, const void* v_host, float scale, void* out_host) {
    if (!ctx) return DC_B200_INVALID_ARGUMENT;
    const bool known = kv && kv->q4 && kv->q4->planned;
    const size_t es = known && kv->q4->type == DC_TYPE_F32 ? 4 : 2, q_bytes = known ? (size_t)kv->q4->T * kv->q4->heads * kv->q4->dim * es : 0;
    auto fail_closed = [&](int st) {
        if (out_host && q_bytes) memset(out_host, 0, q_bytes);
        return st;
    };
    int st = check_call(ctx, kv, layer, "flash_attn_q4");
    if (st != DC_B200_OK) return fail_closed(st);
    if (kv->q4->T == 0) return DC_B200_OK;
    if (!q_host || !out_host || (!k_host != !v_host)) return fail_closed(dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "flash_attn_q4: bad argument"));
    cudaSetDevice(ctx->device);
    const size_t kv_bytes = (size_t)kv->q4->T * kv->q4->kv * kv->q4->dim * es, pad_q = (q_bytes + 255) / 256 * 256, pad_kv = (kv_bytes + 255) / 256 * 256;
    uint8_t* s = dc_scratch(ctx, 2 * pad_q + 2 * pad_kv);
    if (!s) return fail_closed(DC_B200_OUT_OF_MEMORY);
    uint8_t *q = s, *o = s + pad_q, *k = o + pad_q, *v = k + pad_kv;
    auto copy = [&](void* to, const void* from, size_t n, cudaMemcpyKind how) { return dc_check_cuda(ctx, cudaMemcpyAsync(to, from, n, how, ctx->stream), "flash_attn_q4"); };
    st = copy(q, q_host, q_bytes, cudaMemcpyHostToDevice);
    if (st == DC_B200_OK && k_host) st = copy(k, k_host, kv_bytes, cudaMemcpyHostToDevice);
    if (st == DC_B200_OK && k_host) st = copy(v, v_host, kv_bytes, cudaMemcpyHostToDevice);
    if (st == DC_B200_OK) st = dc_b200_flash_attn_q4_dev(ctx, kv, layer, q, 0, k_host ? k : nullptr, k_host ? v : nullptr, 0, scale, o, 0, nullptr, nullptr);
    if (st == DC_B200_OK) st = copy(out_host, o, q_bytes, cudaMemcpyDeviceToHost);
    if (st == DC_B200_OK) st = dc_b200_synchronize(ctx);
    return st == DC_B200_OK ? st : fail_closed(st);
}

int dc_b200_kv_q4_read_block(dc_kv_cache* kv, int layer, int block, float* k_host, float* v_host) {
    if (!kv || !kv->q4 || layer < 0 || layer >= kv->q4->n_layer || block < 0 || block >= kv->max_blocks) return DC_B200_INVALID_ARGUMENT;
    cudaSetDevice(kv->ctx->device);
    const int n_kv = kv->q4->kv, HD = kv->q4->dim, GR = HD / 64, rec = 18 * HD;
    std::vector<uint8_t> page;
    try {
        page.resize((size_t)n_kv * rec);
    } catch (const std::bad_alloc&) {
        return dc_fail(kv->ctx, DC_B200_OUT_OF_MEMORY, "kv_q4_read_block: out of host memory");
    }
    cudaError_t e = cudaStreamSynchronize(kv->ctx->stream);
    if (e == cudaSuccess) e = cudaMemcpy(page.data(), kv->planes[layer].arena + page.size() * block, page.size(), cudaMemcpyDeviceToHost);
    DC_TRY(dc_check_cuda(kv->ctx, e, "kv_q4_read_block"));
    auto half = [&](const uint8_t* at) {
        uint16_t b;
        memcpy(&b, at, 2);
        return __half2float(__ushort_as_half(b));
    };
    for (int tok = 0; tok < DC_KV_BLOCK; ++tok)
        for (int h = 0; h < n_kv; ++h)
            for (int d = 0; d < HD; ++d) {
                const uint8_t* r = page.data() + (size_t)h * rec;
                const int i = d >> 5, t = (d & 7) >> 1, nib = ((d >> 3) & 3) + 4 * (d & 1);
                uint32_t w;
                memcpy(&w, r + (HD == 128 ? dc_q4_rec<128>::k_word(tok, t, i) : dc_q4_rec<64>::k_word(tok, t, i)), 4);
                const uint8_t b = r[HD == 128 ? dc_q4_rec<128>::v_byte(tok, d & 7, d >> 4) : dc_q4_rec<64>::v_byte(tok, d & 7, d >> 4)];
                const uint8_t *ks = r + 8 * HD + (tok * GR + d / 64) * 4, *vs = r + 17 * HD + (tok * GR + d / 64) * 4;
                const size_t to = ((size_t)tok * n_kv + h) * HD + d;
                if (k_host) k_host[to] = fmaf(half(ks), (float)((w >> (4 * nib)) & 15), half(ks + 2));
                if (v_host) v_host[to] = fmaf(half(vs), (float)(d & 8 ? b >> 4 : b & 15), half(vs + 2));
            }
    return DC_B200_OK;
}

}  // extern "C"
