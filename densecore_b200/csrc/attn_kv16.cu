// Attention of a step's new tokens over the paged cache of 16-bit rows whose sequences are kept on the GPU: single tokens, drafted ones, and prompts of f32 rows.
//
//   y = sum_k e^(s q.k - m) v_k / sum_k e^(s q.k - m) over the keys k that a token at position p sees: k <= p and, with a window, k > p - window or k < keep
//
// One pass over the pages with the running maximum and sum.  A warp has 8 NT rows (row r of a sequence: new token r / G, query head r % G of the key head) and takes a page of
// sixteen keys at a time: scores as rows x keys (mma.m16n8k16, queries first), whose accumulators then are the second operand of the answers as dimensions x rows (the
// cache holds values turned), so that no value changes lanes on the way.
//   16-bit rows: queries as they are; f32 rows: queries as two fp16 terms (22 bits) of a row times a power of two, rows h and h + 8 of the operand
//   weights as two terms of the cache's type (bf16 16 bits, fp16 22), so that a result is rounded once; scores, maxima, sums and answers are f32
//   f32 results: a page's answers begin at 0 and are added to the nearest, as the tensor cores' sums are cut off, some 2^-22.7 of themselves an instruction and always towards 0 (one sum over 1875 pages
//   was off by 1.7e-4; 16-bit ones leave it at that: 312 instructions of a warp are 5.6e-5)
// The reference of a row's weights follows its maximum once that is 2^6 ahead: weights up to 64 are as exact, and the answers' factors are rare.  fp16 ends at 2^-25, so its reference lies 2^14
// below the maximum and follows from 2^15 on: a row's weights are off by 2^-22 of themselves or 2^-39 of the largest.  For f32 results, whose second terms are 2^11 fold and have answers of
// their own, by 2^-22 of themselves or 2^-50 of the largest: the rest of a row beside a key that is far ahead of it.
// Work is cut on the GPU, since lengths are there: the pages that all sequences' rows see stand in a line, of which every CTA of a key head takes an equal part; a
// sequence that several CTAs have is joined by the last of them, in the order of its parts, so that results do not depend on who that is.
// Bound: long caches by HBM (48 sequences of up to 32000 positions, bf16, 32 / 4 heads of 128: 1.90 GB in 293 to 305 us, 97 % of a copy's rate); short ones by one chain of loads and barriers, some
// 17 thousand cycles: entries, table, queries and first page, pages, parts, ticket, join (one request of 512 positions 10.1 us, 16 f32 ones of 2300 17.0; 32 requests of 5 fp16 tokens 48.5:
// 9.5, 15.8 and 47.2 while small fp16 weights were lost).  Windows of 1024 over 64 sequences (136 MB)
// 32.5 us: 4.7 TB/s within the pages, the rest is that chain.  Two pages of a warp at a time: one request 9.9 -> 11.6, windows 36 -> 42; four CTAs an SM for heads of 64: 46.6 -> 47.0.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_kv16_tiles.cuh"
#include "dc_launch.cuh"

using namespace dc;

#define DC_TRY(expr)                       \
    do {                                   \
        int _st = (expr);                  \
        if (_st != DC_B200_OK) return _st; \
    } while (0)

namespace {

constexpr int KR_WARPS = 4, KR_SLOTS = 8;      // page places of a CTA, shared out among the groups of warps that take pages in turn
constexpr int KR_LEAST = 16, KR_CTAS = 3;      // pages of a CTA at least (8 to 32: no difference beyond 2 %); CTAs of an SM, as many as shared memory and registers hold

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm4(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename TC>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<TC, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename TC>
struct Two;      // pairs of the cache's type in a word
template <>
struct Two<__half> {
    static constexpr uint32_t EXPONENTS = 0x7C007C00u, ONE = 0x04000400u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};
template <>
struct Two<__nv_bfloat16> {
    static constexpr uint32_t EXPONENTS = 0x7F807F80u, ONE = 0x00800080u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename TX>
__device__ __forceinline__ TX from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

struct RowsParams {
    const dc_kv_entry* entries;
    const int32_t *numbers, *tables;
    int pages_per_seq, heads, n_kv, slots;
    const void *q, *k, *v;      // k null: nothing to write
    int64_t ldq, ldkv, ldo;
    uint8_t* arena;
    float scale;
    int window, keep;
    void* out;
    float* parts;
    int32_t* tickets;
    int part_floats;            // of a part
    bool all;                   // nobody else takes sequences with more rows: one is an error
    const float* prompt_parts;  // of prompt-sized ones, to be added up: k_kv16_prompt of the same call, whose CTAs have begun, is the kernel before (else null)
    int num_sms;
    int* err;
};

template <int HD>
constexpr size_t rows_smem() { return (size_t)KR_SLOTS * dc_kv16_rec<HD>::BYTES + KR_SLOTS * 8 + 1024; }

// The parts of prompt-sized sequences' rows whose keys were split, in their order: a warp per JR rows, a lane HD / 32 dimensions.
template <int HD, typename TX>
__device__ __forceinline__ void join_prompts(const RowsParams& p, int G) {
    constexpr int D = HD / 32, JR = 4;
    const int lane = threadIdx.x & 31;
    const TileLine tiles(p.entries, p.numbers + DC_KV_ENTRIES, p.slots, G, 64, p.n_kv, p.num_sms);
    if (tiles.most == 1) return;
    const size_t step = (size_t)p.n_kv * kp_part_floats<HD>();
    const int warps = gridDim.x * gridDim.y * KR_WARPS, units = tiles.n_all * p.n_kv * (KP_TILE_ROWS / JR);
    for (int x = (blockIdx.y * gridDim.x + blockIdx.x) * KR_WARPS + (threadIdx.x >> 5); x < units; x += warps) {
        const int r0 = x % (KP_TILE_ROWS / JR) * JR, kvh = x / (KP_TILE_ROWS / JR) % p.n_kv, line = x / (KP_TILE_ROWS / JR) / p.n_kv;
        const Tile tl(tiles, line, p.window, p.keep);
        if (tl.n_parts == 1 || r0 >= tl.rows) continue;
        const float* from = p.prompt_parts + ((size_t)line * tiles.most * p.n_kv + kvh) * kp_part_floats<HD>();
        float M[JR], sum[JR], v[JR][D];
#pragma unroll
        for (int b = 0; b < JR; ++b) {
            M[b] = -3e38f, sum[b] = 0.0f;
#pragma unroll
            for (int d = 0; d < D; ++d) v[b][d] = 0.0f;
        }
#pragma unroll 2
        for (int i = 0; i < tl.n_parts; ++i) {
            float2 ml[JR];
            float y[JR][D];
#pragma unroll
            for (int b = 0; b < JR; ++b) {
                const float* at = from + (size_t)i * step + (size_t)min(r0 + b, tl.rows - 1) * (HD + 4);
                ml[b] = __ldcg(reinterpret_cast<const float2*>(at + HD));
                if constexpr (D == 4) {
                    const float4 f = __ldcg(reinterpret_cast<const float4*>(at) + lane);
                    y[b][0] = f.x, y[b][1] = f.y, y[b][2] = f.z, y[b][3] = f.w;
                } else {
                    const float2 f = __ldcg(reinterpret_cast<const float2*>(at) + lane);
                    y[b][0] = f.x, y[b][1] = f.y;
                }
            }
#pragma unroll
            for (int b = 0; b < JR; ++b) {
                const float m = fmaxf(M[b], ml[b].x), f0 = ex2(M[b] - m), f1 = ex2(ml[b].x - m);
                M[b] = m, sum[b] = fmaf(sum[b], f0, ml[b].y * f1);
#pragma unroll
                for (int d = 0; d < D; ++d) v[b][d] = fmaf(v[b][d], f0, y[b][d] * f1);
            }
        }
#pragma unroll
        for (int b = 0; b < JR; ++b) {
            if (r0 + b >= tl.rows) continue;
            const float inv = 1.0f / sum[b];
            const int rr = tl.row0 + r0 + b, j = rr / G;
            TX* to = reinterpret_cast<TX*>(p.out) + (size_t)(tl.e.tok0 + j) * p.ldo + (size_t)(kvh * G + rr - j * G) * HD + D * lane;
            struct alignas(D * sizeof(TX)) Piece {
                TX x[D];
            } y;
#pragma unroll
            for (int d = 0; d < D; ++d) y.x[d] = from_f32<TX>(v[b][d] * inv);
            if (((uintptr_t)to & (sizeof(Piece) - 1)) == 0) {
                *reinterpret_cast<Piece*>(to) = y;
            } else {
#pragma unroll
                for (int d = 0; d < D; ++d) to[d] = y.x[d];
            }
        }
    }
}

// PROMPTS: tiles of 32 NT rows of the sequences that have more, each whole by one CTA; else sequences of up to 32 NT rows, their pages shared out.
template <int HD, typename TX, typename TC, int NT, bool PROMPTS>
__global__ void __launch_bounds__(KR_WARPS * 32, KR_CTAS) k_kv16_rows(const RowsParams p) {
    using R = dc_kv16_rec<HD>;
    using W2 = Two<TC>;
    constexpr bool TERMS = sizeof(TX) == 4;      // queries in two terms
    // The reference of weights lies this many powers of two below a row's maximum where it is taken anew, and follows once the maximum is LAG further ahead
    constexpr float AHEAD = std::is_same<TC, __half>::value ? 14.0f : 0.0f, LAG = std::is_same<TC, __half>::value ? 1.0f : 6.0f;
    static_assert(!std::is_same<TC, __half>::value || AHEAD + LAG <= 15.0f, "weights, and 2^11 times what fp16 leaves of them, are fp16 numbers");
    static_assert(!TERMS || NT == 1, "rows h + 8 of the operand are second terms");
    static_assert(TERMS || !PROMPTS, "prompts of 16-bit rows are k_kv16_prompt's");
    constexpr int RW = 8 * NT, RT = KR_WARPS * RW, KS = HD / 16, VT = HD / 16, PITCH = HD + 4;
    static_assert(KR_WARPS * RW * (PITCH + 2) * 4 <= KR_SLOTS * R::BYTES, "the warps' parts take the pages' place");
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_last;
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t ring = smem_u32(smem), bars = ring + KR_SLOTS * R::BYTES;
    float* part = reinterpret_cast<float*>(smem);      // [warp][RW][PITCH], then maxima and sums [warp][RW][2]
    float* part_ml = part + KR_WARPS * RW * PITCH;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = lane >> 2, t4 = lane & 3, kvh = blockIdx.y, G = p.heads / p.n_kv;
    if (threadIdx.x == 0) {
        for (int s = 0; s < KR_SLOTS; ++s) mbar_init(bars + 8 * s, 1);
        mbar_fence_init();
    }
    __syncthreads();
    // (behind k_kv16_prompt, which has waited for all before it and shares nothing with this one's sequences, the SMs that it leaves idle take them meanwhile)
    if (!p.prompt_parts) pdl_wait();
    pdl_launch_dependents();
    const dc_kv_entry ahead_of = p.entries[min((int)(threadIdx.x & 31), p.slots - 1)];      // (on its way with their number)
    const int n_entries = p.numbers[DC_KV_ENTRIES];
    // ---- the line of work: entries' pages (tiles), a warp of entries at a time
    dc_kv_entry own = {0, 0, 0, 0};
    int chunk = -32, ahead = 0, mine = 0, upto = 0;      // of the chunk's entries: work, and the line's up to with it
    auto weigh = [&](const dc_kv_entry& e) -> int {
        const int rows = e.count * G;      // (at most 2^30, as the whole step's)
        if constexpr (PROMPTS) return rows > RT ? (rows + RT - 1) / RT : 0;
        else return rows <= RT && e.count > 0 ? pages_of(e.pos0, e.pos0 + e.count - 1, p.window, p.keep).n : 0;
    };
    auto look_at = [&](int base) {
        chunk = base;
        own = base + lane >= n_entries ? dc_kv_entry{0, 0, 0, 0} : base == 0 ? ahead_of : p.entries[base + lane];
        mine = weigh(own);
        if (!PROMPTS && p.all && own.count * G > RT) atomicExch(p.err, DC_ERR_STEP);
    };
    int work = 0, n_with = 0;
    for (int base = 0; base < n_entries; base += 32) {
        look_at(base);
        work += mine, n_with += mine > 0;
    }
    work = __reduce_add_sync(0xffffffffu, work), n_with = __reduce_add_sync(0xffffffffu, n_with);
    // Either equal shares of the line, which end within a sequence where they may; or every CTA one part of one sequence, a sequence's parts alike, so that nobody does two
    // chains of loads one after the other: where that leaves no SM with more than 5/4 of the pages (long sequences of unlike lengths keep
    // equal shares).  (All are fewer than 2^31 less the grid's width.)
    const uint32_t ctas = gridDim.x;
    int share = max(KR_LEAST, (int)(((uint32_t)work + ctas - 1) / ctas)), parts = 0;
    bool even = false;
    if (!PROMPTS && n_with < (int)ctas) {
        const int s = max(KR_LEAST, (int)(((uint32_t)work + ctas - n_with - 1) / (ctas - n_with)));      // (with this many pages a part there are no more parts than CTAs)
        int longest = 0;
        for (int base = 0; base < n_entries; base += 32) {
            if (base != chunk) look_at(base);
            const int n = (mine + s - 1) / s;
            parts += n;
            if (n) longest = max(longest, (mine + n - 1) / n);
        }
        parts = __reduce_add_sync(0xffffffffu, parts), longest = __reduce_max_sync(0xffffffffu, longest);
        even = 4 * ((parts * p.n_kv + p.num_sms - 1) / p.num_sms) * longest <= 5 * KR_CTAS * share;
        if (even) share = s;
    }
    int at = PROMPTS || even ? (int)blockIdx.x : (int)min((long long)work, (long long)blockIdx.x * share);
    const int end = PROMPTS ? work : even ? min(at + 1, parts) : min(work, at + share);      // (even: of the parts' line)
    auto begin_line = [&](int base) {
        if (base != chunk) look_at(base);
        upto = even ? (mine + share - 1) / share : mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, s);
            if (lane >= s) upto += o;
        }
        upto += ahead;
    };
    if (at < end) begin_line(0);
    uint32_t phases = 0;      // of the page places
    while (at < end) {
        uint32_t there;
        while (!(there = __ballot_sync(0xffffffffu, upto > at))) {
            ahead = __shfl_sync(0xffffffffu, upto, 31);
            begin_line(chunk + 32);
        }
        const int who = __ffs(there) - 1;
        const int seq = __shfl_sync(0xffffffffu, own.seq, who), pos0 = __shfl_sync(0xffffffffu, own.pos0, who), count = __shfl_sync(0xffffffffu, own.count, who),
                  tok0 = __shfl_sync(0xffffffffu, own.tok0, who);
        const int e_end = __shfl_sync(0xffffffffu, upto, who), e_work = __shfl_sync(0xffffffffu, mine, who), e_parts = even ? (e_work + share - 1) / share : 0, e_at = e_end - (even ? e_parts : e_work);
        // ---- the item: rows from row0 on, pages page0 .. page1 - 1 of those that they see
        const int row0 = PROMPTS ? (at - e_at) * RT : 0, rows = min(RT, count * G - row0), j_last = (row0 + rows - 1) / G;
        const Pages pages = pages_of(pos0 + row0 / G, pos0 + j_last, p.window, p.keep);
        const int e_of = at - e_at, e_each = even ? e_work / e_parts : 0, e_more = even ? e_work - e_each * e_parts : 0;      // (even: part e_of; the first e_more have a page more)
        const int page0 = PROMPTS ? 0 : even ? e_each * e_of + min(e_of, e_more) : e_of;
        const int page1 = PROMPTS ? pages.n : even ? page0 + e_each + (e_of < e_more) : min(end, e_end) - e_at;
        const int tiles = (rows + RW - 1) / RW, lm = tiles <= 1 ? 0 : tiles <= 2 ? 1 : 2, lk = 2 - lm, ld = 3 - lk;      // 2^lm warps share a page, 2^lk groups of them take turns, 2^ld places each
        static_assert(KR_WARPS == 4 && KR_SLOTS == 8, "powers of two");
        const int WM = 1 << lm, WK = 1 << lk, depth = 1 << ld;
        const int grp = warp >> lm, sub = warp & (WM - 1), r0 = row0 + sub * RW, n_my = (page1 - page0 - grp + WK - 1) >> lk;
        const int32_t* table = p.tables + (size_t)seq * p.pages_per_seq;
        auto group_sync = [&]() {
            if (WM == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "r"(32 * WM) : "memory");
        };
        int entry = 0;      // lane i: the page of this group's number i + a multiple of 32
        auto issue = [&](int i, int s) {      // page i of the group's into its place s
            if (i % 32 == 0) entry = i + lane < n_my ? table[pages.at(page0 + grp + ((i + lane) << lk))] : 0;
            const int page = __shfl_sync(0xffffffffu, entry, i % 32);
            if (lane == 0) {
                mbar_expect_tx(bars + 8 * s, R::BYTES);
                bulk_g2s(ring + s * R::BYTES, p.arena + ((size_t)page * p.n_kv + kvh) * R::BYTES, R::BYTES, bars + 8 * s);
            }
        };
        const int s0 = grp << ld;
        auto issue_first = [&]() {
            if (sub == 0)
                for (int i = 0; i < depth && i < n_my; ++i) issue(i, s0 + i);
        };
        // ---- queries: their loads, the table's, the first pages', then what the queries become
        int qpos[NT];
        uint32_t qa[KS][4];
        float F = p.scale * 1.4426950408889634f;
        {
            const TX* src[2];
            bool in[2];
#pragma unroll
            for (int x = 0; x < (TERMS ? 1 : 2); ++x) {
                const int r = r0 + h + 8 * x, j = min(r / G, count - 1);
                in[x] = r < row0 + rows && (x == 0 || NT == 2);
                if (x < NT) qpos[x] = pos0 + j;
                src[x] = reinterpret_cast<const TX*>(p.q) + (size_t)(tok0 + (in[x] ? j : 0)) * p.ldq + (size_t)(kvh * G + (in[x] ? r - j * G : 0)) * HD + 2 * t4;
            }
            if constexpr (TERMS) {
                float x[KS][4], most = 0.0f;
                const bool vec = ((uintptr_t)src[0] & 7) == 0;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float2 f = make_float2(0.0f, 0.0f);
                        if (in[0]) {
                            const float* a = reinterpret_cast<const float*>(src[0]) + 16 * s + 8 * i;
                            if (vec) f = *reinterpret_cast<const float2*>(a);
                            else f = make_float2(a[0], a[1]);
                        }
                        x[s][2 * i] = f.x, x[s][2 * i + 1] = f.y;
                    }
                issue_first();
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(x[s][i]));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // times 2^(10 - e), 2^e <= largest < 2^(e + 1); both factors are normal numbers
                const int e = max(-116, min(127, (int)(__float_as_uint(most) >> 23) - 127));
                const float up = __uint_as_float((uint32_t)(137 - e) << 23);
                F *= __uint_as_float((uint32_t)(117 + e) << 23);
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float a = x[s][2 * i] * up, b = x[s][2 * i + 1] * up;
                        qa[s][2 * i] = W2::pack(a, b);
                        const float2 f = W2::unpack(qa[s][2 * i]);
                        qa[s][2 * i + 1] = W2::pack(a - f.x, b - f.y);
                    }
            } else {
                const bool vec = (((uintptr_t)src[0] | (uintptr_t)src[1]) & 3) == 0;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {      // rows h, h + 8, then eight dimensions on
                        const uint16_t* a = reinterpret_cast<const uint16_t*>(src[i & 1]) + 16 * s + 8 * (i >> 1);
                        qa[s][i] = !in[i & 1] ? 0u : vec ? *reinterpret_cast<const uint32_t*>(a) : a[0] | (uint32_t)a[1] << 16;
                    }
                issue_first();
            }
        }
        // positions between which every row of the warp sees all keys, but for the kept ones
        const int p_least = pos0 + min(r0 / G, count - 1), p_most = pos0 + min((r0 + RW - 1) / G, count - 1), window = p.window ? p.window : 0x7fffffff;
        float o[VT][NT][4], m_run[NT], l[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            m_run[x] = -3.4028235e38f, l[x] = 0.0f;
#pragma unroll
            for (int c = 0; c < VT; ++c) o[c][x][0] = o[c][x][1] = o[c][x][2] = o[c][x][3] = 0.0f;
        }
        const uint32_t k_lane = (lane >> 4) * R::GROUP + (lane & 7) * 128, k_turn = (lane & 7) ^ ((lane >> 3) & 1);
        const uint32_t v_lane = R::VALUES + (lane & 15) * 32 + (((lane >> 4) ^ ((lane >> 2) & 1)) << 4);

        for (int i = 0; i < n_my; ++i) {
            const int s = s0 + (i & (depth - 1)), page = pages.at(page0 + grp + (i << lk)), k0 = page * DC_KV_BLOCK;
            const uint32_t to = ring + s * R::BYTES;
            mbar_wait(bars + 8 * s, ((phases >> s) ^ (i >> ld)) & 1, p.err);
            if (!PROMPTS && p.k && k0 + DC_KV_BLOCK > pos0) {
                // ---- the step's own rows, into the copy and into the cache (no other CTA has this page)
                const int j0 = max(0, k0 - pos0), n = (min(count, k0 + DC_KV_BLOCK - pos0) - j0) * (HD / 2), slot0 = pos0 + j0 - k0;
                uint8_t* rec = p.arena + ((size_t)table[page] * p.n_kv + kvh) * R::BYTES;
                for (int x = sub * 32 + lane; x < n; x += 32 << lm) {
                    const int j = x / (HD / 2), d = 2 * (x % (HD / 2));
                    const size_t from = (size_t)(tok0 + j0 + j) * p.ldkv + (size_t)kvh * HD + d;
                    const TX *ks = reinterpret_cast<const TX*>(p.k) + from, *vs = reinterpret_cast<const TX*>(p.v) + from;
                    const uint32_t kw = W2::pack(to_f32(ks[0]), to_f32(ks[1])), vw = W2::pack(to_f32(vs[0]), to_f32(vs[1]));
                    const uint32_t ka = R::key(slot0 + j, d), va = R::value(slot0 + j, d), vb = R::value(slot0 + j, d + 1);
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + ka), "r"(kw) : "memory");
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + va), "h"((uint16_t)vw) : "memory");
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + vb), "h"((uint16_t)(vw >> 16)) : "memory");
                    *reinterpret_cast<uint32_t*>(rec + ka) = kw;
                    *reinterpret_cast<uint16_t*>(rec + va) = (uint16_t)vw;
                    *reinterpret_cast<uint16_t*>(rec + vb) = (uint16_t)(vw >> 16);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // (a later page is copied here)
                group_sync();
            }
            // ---- scores: c0, c1 of keys 2 t, 2 t + 1 (and eight on) for row h, c2, c3 for row h + 8
            float sc[2][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[0][x] = sc[1][x] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t b[4];
                ldsm4(to + k_lane + ((k_turn ^ ((2 * k) & 7)) << 4) + (k >> 2) * 1024, b);
                mma<TC>(sc[0], qa[k], b[0], b[1]);
                mma<TC>(sc[1], qa[k], b[2], b[3]);
            }
            if constexpr (TERMS) {
#pragma unroll
                for (int a = 0; a < 2; ++a) sc[a][0] += sc[a][2], sc[a][1] += sc[a][3];
            }
            const bool whole = k0 + DC_KV_BLOCK - 1 <= p_least && (k0 > p_most - window || k0 + DC_KV_BLOCK <= p.keep);
            float mx[NT];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int b = 0; b < 2; ++b) sc[a][2 * x + b] *= F;
                if (!whole) {
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int kp = k0 + 8 * a + 2 * t4 + b;
                            if (!(kp <= qpos[x] && (kp > qpos[x] - window || kp < p.keep))) sc[a][2 * x + b] = -INFINITY;
                        }
                }
                mx[x] = fmaxf(fmaxf(sc[0][2 * x], sc[0][2 * x + 1]), fmaxf(sc[1][2 * x], sc[1][2 * x + 1]));
            }
            bool follow = mx[0] > m_run[0] + (AHEAD + LAG);
            if constexpr (NT == 2) follow = follow || mx[1] > m_run[1] + (AHEAD + LAG);
            if (__any_sync(0xffffffffu, follow)) {
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
                    const float m_new = fmaxf(m_run[x], mx[x] - AHEAD), corr = ex2(m_run[x] - m_new);
                    m_run[x] = m_new;
                    l[x] *= corr;
                    const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t4), c1 = __shfl_sync(0xffffffffu, corr, 8 * t4 + 4);
#pragma unroll
                    for (int c = 0; c < VT; ++c) o[c][x][0] *= c0, o[c][x][1] *= c1, o[c][x][2] *= c0, o[c][x][3] *= c1;
                }
            }
            // ---- weights in two terms
            uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const float w0 = ex2(sc[a][2 * x] - m_run[x]), w1 = ex2(sc[a][2 * x + 1] - m_run[x]);
                    l[x] += w0 + w1;
                    hi[x][a] = W2::pack(w0, w1);
                    const float2 f = W2::unpack(hi[x][a]);
                    if constexpr (TERMS) lo[x][a] = W2::pack((w0 - f.x) * 2048.0f, (w1 - f.y) * 2048.0f);
                    else lo[x][a] = W2::pack(w0 - f.x, w1 - f.y);
                }
            // ---- answers.  Where some row does not see some key, a value that is infinite or NaN there must not meet its weight of 0
            uint32_t tops = 0;      // (a half that is infinite or NaN has an exponent of ones: its top bit in the sum with ONE)
            if (!whole) {
#pragma unroll
                for (int c = 0; c < VT; ++c) {
                    uint32_t a[4];
                    ldsm4(to + v_lane + 512 * c, a);
#pragma unroll
                    for (int x = 0; x < 4; ++x) tops |= (a[x] & W2::EXPONENTS) + W2::ONE;
                }
            }
            if (!__any_sync(0xffffffffu, tops & 0x80008000u)) {
#pragma unroll
                for (int c = 0; c < VT; ++c) {
                    uint32_t a[4];
                    ldsm4(to + v_lane + 512 * c, a);
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        if constexpr (TERMS) {      // (a page's own sums, added to the nearest: the tensor cores' sums are cut off)
                            float y[4] = {0.0f, 0.0f, 0.0f, 0.0f}, z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma<TC>(y, a, hi[x][0], hi[x][1]);
                            mma<TC>(z, a, lo[x][0], lo[x][1]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[c][x][i] += fmaf(z[i], 1.0f / 2048.0f, y[i]);
                        } else {
                            mma<TC>(o[c][x], a, hi[x][0], hi[x][1]);
                            mma<TC>(o[c][x], a, lo[x][0], lo[x][1]);
                        }
                    }
                }
            } else {
                // row by row, with the values of the keys that it sees
#pragma unroll 1
                for (int n = 0; n < RW; ++n) {
                    const int x = n >> 3, qp = __shfl_sync(0xffffffffu, x ? qpos[NT - 1] : qpos[0], 4 * (n & 7));
                    uint32_t seen[2];
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        const int kp = k0 + 8 * a + 2 * t4;
                        seen[a] = (kp <= qp && (kp > qp - window || kp < p.keep) ? 0xFFFFu : 0u) | (kp + 1 <= qp && (kp + 1 > qp - window || kp + 1 < p.keep) ? 0xFFFF0000u : 0u);
                    }
                    const uint32_t b[4] = {x ? hi[NT - 1][0] : hi[0][0], x ? hi[NT - 1][1] : hi[0][1], x ? lo[NT - 1][0] : lo[0][0], x ? lo[NT - 1][1] : lo[0][1]};
                    const bool even = (n & 7) == 2 * t4, other = (n & 7) == 2 * t4 + 1;
#pragma unroll
                    for (int c = 0; c < VT; ++c) {
                        uint32_t a[4];
                        ldsm4(to + v_lane + 512 * c, a);
                        a[0] &= seen[0], a[1] &= seen[0], a[2] &= seen[1], a[3] &= seen[1];
                        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        if constexpr (TERMS) {
                            mma<TC>(y, a, b[2], b[3]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[i] *= 1.0f / 2048.0f;
                        }
                        mma<TC>(y, a, b[0], b[1]);
                        if constexpr (!TERMS) mma<TC>(y, a, b[2], b[3]);
#pragma unroll
                        for (int z = 0; z < NT; ++z) {
                            if (z != x) continue;
                            if (even) o[c][z][0] += y[0], o[c][z][2] += y[2];
                            if (other) o[c][z][1] += y[1], o[c][z][3] += y[3];
                        }
                    }
                }
            }
            group_sync();      // the page has been read
            if (sub == 0 && i + depth < n_my) issue(i + depth, s);
        }
        // uses of each place in this item
        for (int g = 0; g < WK; ++g) {
            const int n = (page1 - page0 - g + WK - 1) >> lk;
            for (int s = 0; s < depth; ++s) phases ^= (uint32_t)((n - s + depth - 1) >> ld & 1) << ((g << ld) + s);
        }
        __syncthreads();      // all pages have been read: the parts take their place
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if (t4 == 0) part_ml[2 * (warp * RW + 8 * x + h)] = m_run[x], part_ml[2 * (warp * RW + 8 * x + h) + 1] = l[x];
#pragma unroll
            for (int c = 0; c < VT; ++c) {
                float* at = part + (warp * RW + 8 * x + 2 * t4) * PITCH + 16 * c + h;
                at[0] = o[c][x][0], at[PITCH] = o[c][x][1], at[8] = o[c][x][2], at[PITCH + 8] = o[c][x][3];
            }
        }
        __syncthreads();
        // ---- the groups' parts joined: a thread has four neighbouring dimensions of a row at a time
        const int c_first = PROMPTS ? 0 : even ? e_at : e_at / share, n_parts = PROMPTS ? 1 : even ? e_parts : (e_end - 1) / share - c_first + 1, my_part = PROMPTS ? 0 : (int)blockIdx.x - c_first;
        const bool alone = n_parts == 1;
        auto place = [&](int i) -> float* {      // part i of the sequence
            const int c = c_first + i;
            return p.parts + ((size_t)kvh * 2 * gridDim.x + (i == 0 ? 2 * c + 1 : 2 * c)) * p.part_floats;
        };
        auto store = [&](int r, int d, const float4& v, float inv) {
            const int rr = row0 + r, j = rr / G;
            TX* to = reinterpret_cast<TX*>(p.out) + (size_t)(tok0 + j) * p.ldo + (size_t)(kvh * G + rr - j * G) * HD + d;
            struct alignas(4 * sizeof(TX)) Piece {
                TX x[4];
            } y = {from_f32<TX>(v.x * inv), from_f32<TX>(v.y * inv), from_f32<TX>(v.z * inv), from_f32<TX>(v.w * inv)};
            if (((uintptr_t)to & (sizeof(Piece) - 1)) == 0) *reinterpret_cast<Piece*>(to) = y;
            else to[0] = y.x[0], to[1] = y.x[1], to[2] = y.x[2], to[3] = y.x[3];
        };
        for (int x4 = threadIdx.x; x4 < rows * (HD / 4); x4 += KR_WARPS * 32) {
            const int r = x4 / (HD / 4), d = 4 * (x4 % (HD / 4)), w0 = r / RW, rr = r % RW;
            float M = -3.4028235e38f, L = 0.0f;
            for (int g = 0; g < WK; ++g) M = fmaxf(M, part_ml[2 * (((g << lm) + w0) * RW + rr)]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int g = 0; g < WK; ++g) {
                const int at = ((g << lm) + w0) * RW + rr;
                const float f = ex2(part_ml[2 * at] - M);
                const float4 x = *reinterpret_cast<const float4*>(part + at * PITCH + d);
                L = fmaf(part_ml[2 * at + 1], f, L);
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
            }
            if (alone) {
                store(r, d, v, 1.0f / L);
            } else {
                float* to = place(my_part);
                reinterpret_cast<float4*>(to)[x4] = v;
                if (d == 0) *reinterpret_cast<float2*>(to + RT * HD + 2 * r) = make_float2(M, L);
            }
        }
        if (!alone) {
            int32_t* ticket = p.tickets + (size_t)kvh * gridDim.x + c_first;      // (a CTA is the first of one sequence at most that others have too)
            __syncthreads();
            if (threadIdx.x == 0) {      // (releases what the CTA's threads have stored ahead of the barrier, and acquires what the others' have)
                int before;
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
                s_last = before == n_parts - 1;
                if (s_last) *ticket = 0;
            }
            __syncthreads();
            if (s_last) {
                for (int x4 = threadIdx.x; x4 < rows * (HD / 4); x4 += KR_WARPS * 32) {
                    const int r = x4 / (HD / 4), d = 4 * (x4 % (HD / 4));
                    float M = -3.4028235e38f, L = 0.0f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int B = 8;
                    for (int i0 = 0; i0 < n_parts; i0 += B) {      // eight parts on their way at once
                        float2 ml[B];
                        float4 x[B];
#pragma unroll
                        for (int i = 0; i < B; ++i) {
                            const float* from = place(min(i0 + i, n_parts - 1));
                            ml[i] = __ldcg(reinterpret_cast<const float2*>(from + RT * HD + 2 * r));
                            x[i] = __ldcg(reinterpret_cast<const float4*>(from) + x4);
                        }
                        float m = M;
#pragma unroll
                        for (int i = 0; i < B; ++i) m = fmaxf(m, ml[i].x);
                        const float old = ex2(M - m);
                        M = m, L *= old, v.x *= old, v.y *= old, v.z *= old, v.w *= old;
#pragma unroll
                        for (int i = 0; i < B; ++i) {
                            const float f = i0 + i < n_parts ? ex2(ml[i].x - M) : 0.0f;
                            if (i0 + i < n_parts) L = fmaf(ml[i].y, f, L), v.x = fmaf(x[i].x, f, v.x), v.y = fmaf(x[i].y, f, v.y), v.z = fmaf(x[i].z, f, v.z), v.w = fmaf(x[i].w, f, v.w);
                        }
                    }
                    store(r, d, v, 1.0f / L);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // (the next item's pages are copied where the parts were)
        __syncthreads();
        at = PROMPTS ? at + (int)gridDim.x : min(end, e_end);
    }
    if constexpr (NT == 2 && !PROMPTS) {
        if (p.prompt_parts) {
            pdl_wait();
            join_prompts<HD, TX>(p, G);
        }
    }
}

template <int HD, typename TX, typename TC, int NT, bool PROMPTS>
int launch(dc_ctx* ctx, const dc_kv16_call& c, const RowsParams& p) {
    const auto kernel = k_kv16_rows<HD, TX, TC, NT, PROMPTS>;
    DC_TRY(dc_kernel_setup(ctx, (const void*)kernel, (int)rows_smem<HD>(), "k_kv16_rows"));
    return dc_launch(ctx, "k_kv16_rows", kernel, dim3(dc_kv16_ctas(ctx->num_sms, p.n_kv), p.n_kv), dim3(KR_WARPS * 32), rows_smem<HD>(), p);
}

template <int HD>
int launch_type(dc_ctx* ctx, const dc_kv16_call& c, const RowsParams& p, bool prompts, bool few) {
    const int type = c.kv->dev->type;
    if (type == DC_TYPE_F32) return prompts ? launch<HD, float, __half, 1, true>(ctx, c, p) : launch<HD, float, __half, 1, false>(ctx, c, p);
    if (type == DC_TYPE_F16) return few ? launch<HD, __half, __half, 1, false>(ctx, c, p) : launch<HD, __half, __half, 2, false>(ctx, c, p);
    return few ? launch<HD, __nv_bfloat16, __nv_bfloat16, 1, false>(ctx, c, p) : launch<HD, __nv_bfloat16, __nv_bfloat16, 2, false>(ctx, c, p);
}

}  // namespace

int dc_launch_kv16_rows(dc_ctx* ctx, const dc_kv16_call& c, bool prompts) {
    const dc_kv_dev& z = *c.kv->dev;
    const long long rows = (long long)z.max_count * (z.heads / z.kv);
    const RowsParams p = {z.entries, z.numbers, z.tables, z.pages_per_seq, z.heads, z.kv, z.slots, c.q, c.k, c.v, c.ldq, c.ldkv, c.ldo, c.arena, c.scale, c.window, c.keep, c.out, z.parts, z.tickets,
                          dc_kv16_rows(z.type) * (z.dim + 2), rows <= dc_kv16_rows(z.type), z.type != DC_TYPE_F32 && !prompts && rows > dc_kv16_rows(z.type) ? z.prompt_parts : nullptr,
                          ctx->num_sms, ctx->d_err};
    return z.dim == 128 ? launch_type<128>(ctx, c, p, prompts, rows <= 8) : launch_type<64>(ctx, c, p, prompts, rows <= 8);
}
