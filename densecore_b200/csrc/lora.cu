// Low-rank adapters of many requests beside a shared product: y[t] = base[t] + s_a (x[t] A_a^T) B_a^T with a = ids[t], rows of other ids (none, unknown, empty)
// y[t] = base[t].  Two kernels: h = s x A^T, then y = base + h B^T.
// Few rows: a warp per rank of a row, then a thread per column of a row; what counts is the number of loads that wait for one another (id, rank, matrix), and
// every matrix row is in flight at once.  Many rows: tiles of rows on the tensor cores.
//
// Tiles: rows x and h are f32 and enter the tensor cores as two terms of 11 bits (tf32, 22 bits together; products of m16n8k8 with f32 sums), matrices are bf16 or
// fp16, which tf32 holds exactly.  A tile whose rows have several adapters takes one after the other: each
// adapter's matrices are read once per tile, whatever the order of rows; up to 256 rows are put in their adapters' order first.
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_launch.cuh"

using namespace dc;

#define DC_TRY(expr)                       \
    do {                                   \
        int _st = (expr);                  \
        if (_st != DC_B200_OK) return _st; \
    } while (0)

struct dc_lora {
    dc_ctx* ctx = nullptr;
    int64_t K = 0, N = 0, Kp = 0, Np = 0;      // padded to 16 and 8
    int slots = 0, max_rank = 0, Rp = 0, type = 0;      // ranks padded to 16
    uint16_t *a = nullptr, *b = nullptr;      // [slot][Rp][Kp] and [slot][Np][Rp], zero where there is nothing
    int32_t* rank = nullptr;                  // [slot], 0: empty
    float* scale = nullptr;
    float* h = nullptr;                       // workspace [parts][rows][Rp]
    int64_t h_rows = 0;
    int32_t* order = nullptr;                 // workspace of k_lora_order
    std::vector<float*> retired;              // outgrown workspaces, which captured calls may still name
};

namespace {

struct LoraParams {
    const uint16_t *a, *b;
    const int32_t* rank;
    const float* scale;
    int slots, Rp;
    int64_t K, N, Kp, Np;
    const float* x;
    int64_t ldx;
    int M;
    const int32_t* ids;
    float* h;
    const float* base;
    float* y;
    int64_t ldb, ldy;
    const int32_t* order;      // rows by adapter (k_lora_order), or NULL: as they come
};

__device__ __forceinline__ int slot_of(const LoraParams& p, int row) {      // -1: none
    if (row >= p.M) return -1;
    const int a = p.ids[row];
    return a >= 0 && a < p.slots && p.rank[a] > 0 ? a : -1;
}
// Tiles: place i of all rows has row row_at(i); h is held by places
__device__ __forceinline__ int row_at(const LoraParams& p, int i) { return i < p.M ? (p.order ? p.order[i] : i) : p.M; }
template <bool BF>
__device__ __forceinline__ float2 two(uint32_t w) {
    if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The product of 16 neighbours along k: lane (h, t) holds rows h, h + 8 of the first operand and column h of the second, k = 4 t .. 4 t + 3.  Two steps of
// k8 (4 t and 4 t + 1 stand for t and t + 4 of the first, 4 t + 2 and 4 t + 3 of the second), the low terms first.
struct Terms {
    uint32_t hi[2][4], lo[2][4];
    __device__ __forceinline__ Terms(const float4& u, const float4& v) {
        const float r[2][4] = {{u.x, u.y, u.z, u.w}, {v.x, v.y, v.z, v.w}};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {      // rows h, h + 8 at k = t, then at t + 4
                const float f = r[i & 1][2 * s + (i >> 1)];
                hi[s][i] = __float_as_uint(f) & 0xFFFFE000u;
                lo[s][i] = __float_as_uint(f - __uint_as_float(hi[s][i]));
            }
    }
    __device__ __forceinline__ void times(float (&d)[4], const float2& b01, const float2& b23) const {
        mma_tf32(d, lo[0], __float_as_uint(b01.x), __float_as_uint(b01.y));
        mma_tf32(d, lo[1], __float_as_uint(b23.x), __float_as_uint(b23.y));
        mma_tf32(d, hi[0], __float_as_uint(b01.x), __float_as_uint(b01.y));
        mma_tf32(d, hi[1], __float_as_uint(b23.x), __float_as_uint(b23.y));
    }
};
__device__ __forceinline__ float4 load_x4(const float* row, int64_t k, int64_t K, bool vec, bool in) {
    if (!in || k >= K) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec && k + 4 <= K) return __ldg(reinterpret_cast<const float4*>(row + k));
    return make_float4(row[k], k + 1 < K ? row[k + 1] : 0.f, k + 2 < K ? row[k + 2] : 0.f, k + 3 < K ? row[k + 3] : 0.f);
}

// Few rows: a warp per rank of a row.  Bound: three loads that wait for one another; with k_lora_up_rows 6.4 us for a row (K 2048, N 5120, rank 16), 9.3 for 64 of rank 32.
template <bool BF>
__global__ void __launch_bounds__(256) k_lora_down(const LoraParams p, int vec) {
    const int row = blockIdx.x, r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    const int a = slot_of(p, row);
    if (a < 0 || r >= (p.rank[a] + 15) / 16 * 16) return;      // (the padding's rows of the matrix are zero, so are its sums)
    const uint16_t* w = p.a + ((size_t)a * p.Rp + r) * p.Kp;
    const float* x = p.x + (size_t)row * p.ldx;
    const float scale = p.scale[a];
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll 8
    for (int64_t k = 8 * lane; k < p.Kp; k += 256) {
        const uint4 c = __ldg(reinterpret_cast<const uint4*>(w + k));
        const float4 u = load_x4(x, k, p.K, vec, true), v = load_x4(x, k + 4, p.K, vec, true);
        const float2 c0 = two<BF>(c.x), c1 = two<BF>(c.y), c2 = two<BF>(c.z), c3 = two<BF>(c.w);
        s0 = fmaf(u.x, c0.x, s0), s1 = fmaf(u.y, c0.y, s1), s0 = fmaf(u.z, c1.x, s0), s1 = fmaf(u.w, c1.y, s1);
        s0 = fmaf(v.x, c2.x, s0), s1 = fmaf(v.y, c2.y, s1), s0 = fmaf(v.z, c3.x, s0), s1 = fmaf(v.w, c3.y, s1);
    }
    s0 += s1;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, s);
    if (lane == 0) p.h[(size_t)row * p.Rp + r] = s0 * scale;
}

// Few rows: a thread per column of a row, sixteen ranks (two loads of its row of the matrix) at a time.
template <bool BF>
__global__ void __launch_bounds__(128) k_lora_up_rows(const LoraParams p) {
    const int row = blockIdx.y;
    const int64_t n = (int64_t)blockIdx.x * 128 + threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    if (n >= p.N) return;
    const int a = slot_of(p, row);
    float sum = p.base[(size_t)row * p.ldb + n], add = 0.0f;
    if (a >= 0) {
        const int ranks = p.rank[a];
        const uint16_t* w = p.b + ((size_t)a * p.Np + n) * p.Rp;
        const float* h = p.h + (size_t)row * p.Rp;
#pragma unroll 2
        for (int r = 0; r < ranks; r += 16) {
            const uint4 c[2] = {__ldg(reinterpret_cast<const uint4*>(w + r)), __ldg(reinterpret_cast<const uint4*>(w + r + 8))};
            float4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __ldcg(reinterpret_cast<const float4*>(h + r) + i);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 c0 = two<BF>(c[i].x), c1 = two<BF>(c[i].y), c2 = two<BF>(c[i].z), c3 = two<BF>(c[i].w);
                add = fmaf(u[2 * i].x, c0.x, add), add = fmaf(u[2 * i].y, c0.y, add), add = fmaf(u[2 * i].z, c1.x, add), add = fmaf(u[2 * i].w, c1.y, add);
                add = fmaf(u[2 * i + 1].x, c2.x, add), add = fmaf(u[2 * i + 1].y, c2.y, add), add = fmaf(u[2 * i + 1].z, c3.x, add), add = fmaf(u[2 * i + 1].w, c3.y, add);
            }
        }
    }
    p.y[(size_t)row * p.ldy + n] = sum + add;
}

// Rows by adapter, those without one last, else as they come: a row's place is the number of rows before it.  One CTA, some 5 us with its launch.
// A tile of several adapters takes a pass for each: 200 mixed rows of rank 64 40 us as they come, 27 in order; runs, as prompts have them, gain nothing by an order, 22 and 28 us
// at 384 rows.  Above 256 rows they are taken as they come, right for runs and slow for mixed rows (K 2048, N 6144, rank 64): 300 rows of 4 adapters 18 us in runs, 43 mixed,
// of 48 21 and 135; 2011 rows 66 and 175, 70 and 484.
constexpr int LORA_SORTED = 256;
__global__ void __launch_bounds__(LORA_SORTED) k_lora_order(const LoraParams p, int32_t* order) {
    __shared__ __align__(16) int slot[LORA_SORTED];
    const int i = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const int a = slot_of(p, i), mine = a < 0 ? 0x7fffffff : a;
    slot[i] = mine;      // (places from M on count for nobody: none, and behind all)
    __syncthreads();
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < (p.M + 3) / 4; ++j) {
        const int4 s = *reinterpret_cast<const int4*>(slot + 4 * j);
        place += (s.x < mine || (s.x == mine && 4 * j < i)) + (s.y < mine || (s.y == mine && 4 * j + 1 < i)) + (s.z < mine || (s.z == mine && 4 * j + 2 < i)) +
                 (s.w < mine || (s.w == mine && 4 * j + 3 < i));
    }
    if (i < p.M) order[place] = i;
}

// Adapters of a tile's rows, one after the other: `f(slot, mask)` with the rows (bits) that have it.
template <typename F>
__device__ __forceinline__ void each_adapter(int mine, uint32_t rows, F f) {      // mine: lane i's row's slot; rows: bits to look at
    uint32_t todo = __ballot_sync(0xffffffffu, mine >= 0) & rows;
    while (todo) {
        const int a = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
        const uint32_t mask = __ballot_sync(0xffffffffu, mine == a) & rows;
        f(a, mask);
        todo &= ~mask;
    }
}

// A row's sums are stored by its own adapter's pass; the others' may leave anything there (zero times an infinite matrix).
// Many rows: a CTA per (16 rows, 8 NT ranks, part of k), its warps share out the part in steps of 16 and add up in the end; the parts are added by the next kernel.
// Bound: latency of one part's loads and sums (17 us of 2011 rows, K 2048, rank 64), and tiles with the rows of two adapters, which take two passes.  Sixteen ranks leave registers for
// eight steps' loads at once, 32 for four: 746 rows, K 7408, N 2656, rank 2 by 16 ranks 28 us, by 64 (two steps) 45; rank 64 by 32 ranks 44, by 64 54, by 16 50.
template <bool BF, int NT>
__global__ void __launch_bounds__(256, 2) k_lora_down_tile(const LoraParams p, int vec) {
    constexpr int DT_R = 8 * NT;
    __shared__ float part[8][16][DT_R + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = lane >> 2, t = lane & 3, row0 = blockIdx.x * 16, r0 = blockIdx.y * DT_R;
    pdl_wait();
    pdl_launch_dependents();
    const int mine = slot_of(p, row_at(p, row0 + (lane & 15)));
    const int row_u = row_at(p, row0 + h), row_v = row_at(p, row0 + h + 8);
    const int64_t per = (p.Kp / 16 + gridDim.z - 1) / gridDim.z * 16, k0 = blockIdx.z * per, k1 = min(p.Kp, k0 + per);
    each_adapter(mine, 0xFFFFu, [&](int a, uint32_t mask) {      // (the same ones in all warps)
        const int tiles = min(NT, ((p.rank[a] + 15) / 16 * 16 - r0) / 8);
        if (tiles <= 0) return;
        const float scale = p.scale[a];
        float sum[NT][4] = {};
        const bool u = mask >> h & 1, v = mask >> (h + 8) & 1;
        const float *xu = p.x + (size_t)(u ? row_u : 0) * p.ldx, *xv = p.x + (size_t)(v ? row_v : 0) * p.ldx;
        const uint16_t* w = p.a + ((size_t)a * p.Rp + r0 + h) * p.Kp + 4 * t;
#pragma unroll (16 / NT)
        for (int64_t k = k0 + 16 * warp; k < k1; k += 128) {
            uint2 c[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) c[i] = i < tiles ? __ldg(reinterpret_cast<const uint2*>(w + (size_t)(8 * i) * p.Kp + k)) : make_uint2(0, 0);
            const Terms x(load_x4(xu, k + 4 * t, p.K, vec, u), load_x4(xv, k + 4 * t, p.K, vec, v));
#pragma unroll
            for (int i = 0; i < NT; ++i)
                if (i < tiles) x.times(sum[i], two<BF>(c[i].x), two<BF>(c[i].y));
        }
        __syncthreads();      // (the last adapter's sums have been read)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            part[warp][h][8 * i + 2 * t] = sum[i][0], part[warp][h][8 * i + 2 * t + 1] = sum[i][1];
            part[warp][h + 8][8 * i + 2 * t] = sum[i][2], part[warp][h + 8][8 * i + 2 * t + 1] = sum[i][3];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * DT_R; i += 256) {
            const int row = i / DT_R, r = i % DT_R;
            if (!(mask >> row & 1) || r >= 8 * tiles) continue;
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) s += part[q][row][r];
            p.h[((size_t)blockIdx.z * p.M + row0 + row) * p.Rp + r0 + r] = s * scale;
        }
    });
}

// Many rows: y = base + h B^T, a CTA per (16 rows, 256 columns), a warp has 32 columns.  h comes in `parts` sums, 128 ranks of it at a time; base is on its way
// meanwhile.  Bound: base and y, and the two-term products beside them: 2011 rows, N 6144, K 2048, rank 64: some 45 of the call's 61 to 68 us, 2.2 TB/s; base and y without products would
// take 22.  (Several tiles a CTA with the matrix in shared memory and base fetched three tiles ahead: 73 us a call where this took 70; two CTAs an SM with more
// loads on their way 74 against 68; four with 64 registers spill: 78.)
constexpr int UP_R = 128;
template <bool BF>
__global__ void __launch_bounds__(256, 3) k_lora_up(const LoraParams p, int vec, int parts) {
    constexpr int MT = 1, NP = 4;
    __shared__ __align__(16) float sh[16 * MT][UP_R + 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = lane >> 2, t = lane & 3, row0 = blockIdx.y * 16 * MT;
    const int64_t n0 = ((int64_t)blockIdx.x * 8 + warp) * 8 * NP;
    pdl_wait();
    pdl_launch_dependents();
    const int rows[2] = {row_at(p, row0 + h), row_at(p, row0 + h + 8)};
    float2 f[2][NP];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int row = rows[q];
        const float* from = p.base + (size_t)(row < p.M ? row : 0) * p.ldb;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int64_t n = n0 + 8 * i + 2 * t;
            if (vec && n + 1 < p.N) f[q][i] = *reinterpret_cast<const float2*>(from + n);
            else f[q][i] = make_float2(n < p.N ? from[n] : 0.f, n + 1 < p.N ? from[n + 1] : 0.f);
        }
    }
    const int mine = slot_of(p, row_at(p, row0 + (lane & 15)));
    auto store = [&](const float (&sum)[MT][NP][4], uint32_t mask) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (!(mask >> (h + 8 * q) & 1)) continue;
            float* to = p.y + (size_t)rows[q] * p.ldy;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int64_t n = n0 + 8 * i + 2 * t;
                const float2 v = make_float2(f[q][i].x + sum[0][i][2 * q], f[q][i].y + sum[0][i][2 * q + 1]);
                if (vec && n + 1 < p.N) {
                    *reinterpret_cast<float2*>(to + n) = v;
                } else {
                    if (n < p.N) to[n] = v.x;
                    if (n + 1 < p.N) to[n + 1] = v.y;
                }
            }
        }
    };
    uint32_t rest = p.M - row0 >= 16 ? 0xFFFFu : (1u << (p.M - row0)) - 1u;
    each_adapter(mine, rest, [&](int a, uint32_t mask) {      // (the same ones in all warps)
        const int ranks = (p.rank[a] + 15) / 16 * 16;
        const uint16_t* w = p.b + ((size_t)a * p.Np + n0 + h) * p.Rp + 4 * t;
        float sum[MT][NP][4] = {};
        for (int r0 = 0; r0 < ranks; r0 += UP_R) {
            const int here = min(UP_R, ranks - r0), per = here / 4;
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * MT * per; i += 256) {
                const int row = i / per, c = i - row * per;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (mask >> row & 1)
#pragma unroll 4
                    for (int z = 0; z < parts; ++z) {
                        const float4 o = __ldcg(reinterpret_cast<const float4*>(p.h + ((size_t)z * p.M + row0 + row) * p.Rp + r0) + c);
                        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
                    }
                *reinterpret_cast<float4*>(&sh[row][4 * c]) = v;
            }
            __syncthreads();
#pragma unroll 4
            for (int r = 0; r < here; r += 16) {
                uint2 c[NP];
#pragma unroll
                for (int i = 0; i < NP; ++i) c[i] = n0 + 8 * i < p.Np ? __ldg(reinterpret_cast<const uint2*>(w + (size_t)(8 * i) * p.Rp + r0 + r)) : make_uint2(0, 0);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (!(mask >> (16 * m) & 0xFFFFu)) continue;
                    const Terms x(*reinterpret_cast<const float4*>(&sh[16 * m + h][r + 4 * t]), *reinterpret_cast<const float4*>(&sh[16 * m + h + 8][r + 4 * t]));
#pragma unroll
                    for (int i = 0; i < NP; ++i) x.times(sum[m][i], two<BF>(c[i].x), two<BF>(c[i].y));
                }
            }
        }
        store(sum, mask);
        rest &= ~mask;
    });
    if (rest && (p.y != p.base || p.ldy != p.ldb)) {      // rows without an adapter
        const float none[MT][NP][4] = {};
        store(none, rest);
    }
}

// One adapter's matrices into their padded places; `rank` 0 empties the slot.
__global__ void __launch_bounds__(256) k_lora_set(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b, uint16_t* __restrict__ to_a, uint16_t* __restrict__ to_b, int rank, int Rp,
                                                  int64_t K, int64_t Kp, int64_t N, int64_t Np, int32_t* rank_at, float* scale_at, float scale) {
    pdl_wait();
    const int64_t all_a = (int64_t)Rp * Kp, all = all_a + Np * Rp;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        if (i < all_a) {
            const int64_t r = i / Kp, k = i - r * Kp;
            to_a[i] = r < rank && k < K ? a[r * K + k] : (uint16_t)0;
        } else {
            const int64_t n = (i - all_a) / Rp, r = (i - all_a) - n * Rp;
            to_b[i - all_a] = r < rank && n < N ? b[n * rank + r] : (uint16_t)0;
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *rank_at = rank, *scale_at = scale;
}

// Rows from which tiles are taken: they read a matrix once for 16 rows of one adapter; below, one warp a rank and one thread a column have shorter chains of loads.
// K 2048, N 6144, four adapters mixed, by rows and by tiles of rows in order, in us: 100 rows of rank 32 13 and 21, 256 22 and 25; 100 rows of rank 64 25 and 23, 256 49 and 28;
// rank 128 42 and 27, 87 and 34.
int tile_rows(int Rp) { return Rp <= 32 ? 257 : 97; }
constexpr int LORA_PARTS = 8;      // of k, at most

// Until the CTAs fill the SMs three times, a warp keeping two steps, and four from the fifth part on: 400 rows, K 8192, rank 16 in four parts 17.8 us, in eight 15.9; 700 rows, K 2048,
// rank 64 30.5 and 32.5.
int parts_of(const dc_ctx* ctx, int M, int64_t Kp) {
    int n = 1;
    while (n < LORA_PARTS && (M + 15) / 16 * n < 3 * ctx->num_sms && Kp / (16 * 8 * 2 * n) >= (n < 4 ? 2 : 4)) n *= 2;
    return n;
}

template <bool BF>
int launch_add(dc_ctx* ctx, LoraParams p, int max_rank, int32_t* order) {
    const int vx = ((uintptr_t)p.x & 15) == 0 && p.ldx % 4 == 0, vy = ((uintptr_t)p.base & 7) == 0 && ((uintptr_t)p.y & 7) == 0 && p.ldb % 2 == 0 && p.ldy % 2 == 0;
    if (p.M < tile_rows(p.Rp)) {
        DC_TRY(dc_launch(ctx, "k_lora_down", k_lora_down<BF>, dim3(p.M, (max_rank + 15) / 16 * 2), dim3(256), 0, p, vx));
        return dc_launch(ctx, "k_lora_up_rows", k_lora_up_rows<BF>, dim3((unsigned)((p.N + 127) / 128), p.M), dim3(128), 0, p);
    }
    const int parts = parts_of(ctx, p.M, p.Kp);
    p.order = nullptr;
    if (p.M <= LORA_SORTED) {
        DC_TRY(dc_launch(ctx, "k_lora_order", k_lora_order, dim3(1), dim3(LORA_SORTED), 0, p, order));
        p.order = order;
    }
    const int ranks = p.Rp <= 16 ? 16 : 32;      // of a CTA
    auto down = ranks == 16 ? k_lora_down_tile<BF, 2> : k_lora_down_tile<BF, 4>;
    DC_TRY(dc_launch(ctx, "k_lora_down_tile", down, dim3((p.M + 15) / 16, (p.Rp + ranks - 1) / ranks, parts), dim3(256), 0, p, vx));
    return dc_launch(ctx, "k_lora_up", k_lora_up<BF>, dim3((unsigned)((p.N + 255) / 256), (p.M + 15) / 16), dim3(256), 0, p, vy, parts);
}

int grow(dc_ctx* ctx, dc_lora* l, int64_t rows) {
    if (rows <= l->h_rows) return DC_B200_OK;
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(ctx->stream, &st) == cudaSuccess && st != cudaStreamCaptureStatusNone)
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "lora_add: the first call with %lld rows or more cannot be captured", (long long)rows);
    float* fresh = nullptr;
    const int64_t want = std::max<int64_t>(rows + rows / 2, 64);
    DC_TRY(dc_check_cuda(ctx, cudaMalloc(&fresh, (size_t)want * l->Rp * 4), "lora workspace"));
    try {
        if (l->h) l->retired.push_back(l->h);
    } catch (const std::bad_alloc&) {
        cudaFree(fresh);
        return dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "lora workspace: out of host memory");
    }
    l->h = fresh, l->h_rows = want;
    return DC_B200_OK;
}

constexpr int LORA_ROWS = 65535 * 16;      // of a call: a grid's second dimension

// Room for the row sums of a call of M rows.
int make_room(dc_ctx* ctx, dc_lora* l, int M) { return grow(ctx, l, M < tile_rows(l->Rp) ? M : (int64_t)M * parts_of(ctx, M, l->Kp)); }

int check_set(dc_lora* l, int slot, int rank, const void* a, const void* b, float scale) {
    if (slot < 0 || slot >= l->slots || rank < 0 || rank > l->max_rank || (rank && (!a || !b)) || !isfinite(scale))
        return dc_fail(l->ctx, DC_B200_INVALID_ARGUMENT, "lora_set: slot %d of %d, rank %d of at most %d", slot, l->slots, rank, l->max_rank);
    return DC_B200_OK;
}

void release(dc_lora* l) {      // (what it does not have is null)
    cudaFree(l->a), cudaFree(l->b), cudaFree(l->rank), cudaFree(l->scale), cudaFree(l->order), cudaFree(l->h);
    for (float* h : l->retired) cudaFree(h);
    delete l;
}

}  // namespace

extern "C" {

int dc_b200_lora_create(dc_ctx* ctx, int64_t K, int64_t N, int max_adapters, int max_rank, int type, dc_lora** out) {
    if (!ctx || !out) return DC_B200_INVALID_ARGUMENT;
    *out = nullptr;
    if (K < 1 || N < 1 || K > (1 << 24) || N > (1 << 24) || max_adapters < 1 || max_rank < 1 || max_rank > 4096)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "lora_create: bad shape (%lld x %lld, %d adapters of rank %d)", (long long)K, (long long)N, max_adapters, max_rank);
    if (type != DC_TYPE_BF16 && type != DC_TYPE_F16) return dc_fail(ctx, DC_B200_UNSUPPORTED, "lora_create: matrices of type %d (BF16 and F16 are supported)", type);
    // (2^40 numbers a matrix are beyond any device's memory, and their bytes clear of 64 bits' end)
    if (max_adapters > (int64_t(1) << 40) / ((max_rank + 15) / 16 * 16 * (std::max(K, N) + 15)))
        return dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "lora_create: %d adapters of rank %d beside a matrix of %lld x %lld", max_adapters, max_rank, (long long)N, (long long)K);
    cudaSetDevice(ctx->device);
    dc_lora* l = new (std::nothrow) dc_lora();
    if (!l) return dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "lora_create: out of host memory");
    l->ctx = ctx, l->K = K, l->N = N, l->Kp = (K + 15) / 16 * 16, l->Np = (N + 7) / 8 * 8;
    l->slots = max_adapters, l->max_rank = max_rank, l->Rp = (max_rank + 15) / 16 * 16, l->type = type;
    cudaError_t e = cudaMalloc(&l->a, (size_t)max_adapters * l->Rp * l->Kp * 2);
    if (e == cudaSuccess) e = cudaMalloc(&l->b, (size_t)max_adapters * l->Np * l->Rp * 2);
    if (e == cudaSuccess) e = cudaMalloc(&l->rank, (size_t)max_adapters * 4);
    if (e == cudaSuccess) e = cudaMalloc(&l->order, LORA_SORTED * 4);
    if (e == cudaSuccess) e = cudaMalloc(&l->scale, (size_t)max_adapters * 4);
    if (e == cudaSuccess) e = cudaMemsetAsync(l->rank, 0, (size_t)max_adapters * 4, ctx->stream);
    if (e != cudaSuccess) {
        const int st = dc_check_cuda(ctx, e, "lora_create");
        release(l);
        return st;
    }
    *out = l;
    return DC_B200_OK;
}

void dc_b200_lora_destroy(dc_lora* l) {
    if (!l) return;
    cudaSetDevice(l->ctx->device);
    cudaStreamSynchronize(l->ctx->stream);
    release(l);
}

int dc_b200_lora_set_dev(dc_lora* l, int slot, int rank, const void* a_dev, const void* b_dev, float scale) {
    if (!l) return DC_B200_INVALID_ARGUMENT;
    DC_TRY(check_set(l, slot, rank, a_dev, b_dev, scale));
    dc_ctx* ctx = l->ctx;
    cudaSetDevice(ctx->device);
    const int64_t all = (int64_t)l->Rp * (l->Kp + l->Np);
    return dc_launch(ctx, "k_lora_set", k_lora_set, dim3((unsigned)std::min<int64_t>((all + 255) / 256, ctx->num_sms * 16)), dim3(256), 0, (const uint16_t*)a_dev, (const uint16_t*)b_dev,
                     l->a + (size_t)slot * l->Rp * l->Kp, l->b + (size_t)slot * l->Np * l->Rp, rank, l->Rp, l->K, l->Kp, l->N, l->Np, l->rank + slot, l->scale + slot, scale);
}

int dc_b200_lora_set(dc_lora* l, int slot, int rank, const void* a_host, const void* b_host, float scale) {
    if (!l) return DC_B200_INVALID_ARGUMENT;
    DC_TRY(check_set(l, slot, rank, a_host, b_host, scale));
    dc_ctx* ctx = l->ctx;
    cudaSetDevice(ctx->device);
    const size_t na = (size_t)rank * l->K * 2, nb = (size_t)rank * l->N * 2, pad = (na + 255) / 256 * 256;
    uint8_t* s = dc_scratch(ctx, pad + nb + 256);
    if (!s) return DC_B200_OUT_OF_MEMORY;
    if (rank) DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(s, a_host, na, cudaMemcpyHostToDevice, ctx->stream), "lora_set"));
    if (rank) DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(s + pad, b_host, nb, cudaMemcpyHostToDevice, ctx->stream), "lora_set"));
    DC_TRY(dc_b200_lora_set_dev(l, slot, rank, s, s + pad, scale));
    return dc_b200_synchronize(ctx);
}

int dc_b200_lora_add_dev(dc_ctx* ctx, dc_lora* l, const float* x_dev, int64_t ld_x, int M, const int32_t* ids_dev, const float* base_dev, int64_t ld_base, float* y_dev, int64_t ld_y) {
    if (!ctx || !l) return DC_B200_INVALID_ARGUMENT;
    if (l->ctx != ctx) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "lora_add: the adapters belong to another context");
    if (ld_x == 0) ld_x = l->K;
    if (ld_base == 0) ld_base = l->N;
    if (ld_y == 0) ld_y = l->N;
    if (M < 0 || M > LORA_ROWS || ld_x < l->K || ld_base < l->N || ld_y < l->N)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "lora_add: bad argument (%d rows, strides %lld, %lld, %lld)", M, (long long)ld_x, (long long)ld_base, (long long)ld_y);
    if (M == 0) return DC_B200_OK;
    if (!x_dev || !ids_dev || !y_dev) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "lora_add: null buffer");
    if (!base_dev) base_dev = y_dev, ld_base = ld_y;
    cudaSetDevice(ctx->device);
    DC_TRY(make_room(ctx, l, M));
    const LoraParams p = {l->a, l->b, l->rank, l->scale, l->slots, l->Rp, l->K, l->N, l->Kp, l->Np, x_dev, ld_x, M, ids_dev, l->h, base_dev, y_dev, ld_base, ld_y, nullptr};
    return l->type == DC_TYPE_BF16 ? launch_add<true>(ctx, p, l->max_rank, l->order) : launch_add<false>(ctx, p, l->max_rank, l->order);
}

int dc_b200_mul_mat_lora_dev(dc_ctx* ctx, const dc_weight* w, dc_lora* l, const float* x_dev, int M, const int32_t* ids_dev, float* y_dev) {
    if (!ctx || !w || !l) return DC_B200_INVALID_ARGUMENT;
    if (w->K != l->K || w->N != l->N || w->E != 1)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "mul_mat_lora: adapters of %lld x %lld beside a matrix of %lld x %lld", (long long)l->K, (long long)l->N, (long long)w->K, (long long)w->N);
    if (M < 1 || M > LORA_ROWS || !x_dev || !ids_dev || !y_dev) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "mul_mat_lora: bad argument (%d rows)", M);
    const uintptr_t x0 = (uintptr_t)x_dev, x1 = (uintptr_t)(x_dev + (size_t)M * l->K), y0 = (uintptr_t)y_dev, y1 = (uintptr_t)(y_dev + (size_t)M * l->N);
    if (!(x1 <= y0 || y1 <= x0)) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "mul_mat_lora: x and y overlap");
    if (l->ctx != ctx) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "mul_mat_lora: the adapters belong to another context");
    cudaSetDevice(ctx->device);
    DC_TRY(make_room(ctx, l, M));      // (ahead of the product: a refused call has enqueued nothing)
    DC_TRY(dc_b200_mul_mat_dev(ctx, w, x_dev, M, y_dev));
    return dc_b200_lora_add_dev(ctx, l, x_dev, 0, M, ids_dev, nullptr, 0, y_dev, 0);
}

}  // extern "C"
