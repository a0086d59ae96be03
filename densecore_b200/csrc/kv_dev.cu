// Sequences of a paged cache kept on the GPU: lengths, pages and block tables change by a kernel, so that a step can follow the one whose result it depends on (how
// many drafted tokens were accepted) without the host, and a run of steps fits into one CUDA graph.
//
// Every slot s holds held[s] pages for lens[s] tokens.  A step takes its last `drop` tokens from it and asks for `count` new ones:
//   keep = len - min(max(drop, 0), len), need = ceil((keep + count) / 16); it frees what it holds beyond need, or asks for what is missing.
// Free pages are a stack F[0 .. n).  With R pages freed and A granted, all in the order of slots and places, the j-th granted one is the j-th freed one, or
// F[n - 1 - (j - R)] behind those; what is left of the freed ones goes onto the stack in falling order.  So a step and the one that takes it back leave the
// tables and the stack as they were.
// All of it is prefix sums over the slots (k_kv_step, one CTA, or each CTA of a cluster for itself: a slot's numbers are some bytes), behind which every page that new
// tokens lie on is a unit of work of its own: it is looked up or granted, and its tokens' places are written.  The largest steps share the units out among all SMs
// (k_kv_places).
// Bound: latency of a launch, the loads and two scans (5 us a step of 16 sequences); the largest steps by their tokens' twelve bytes and by the chain of a unit, page, token.  A step of 512
// sequences that brings two million tokens (up to 8192 each) or takes them back: 13 us, 4 of them its floor at the rate of a copy.
#include <cooperative_groups.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "dc_common.cuh"
#include "dc_internal.h"
#include "dc_kv_dev.h"
#include "dc_launch.cuh"

namespace cg = cooperative_groups;
using namespace dc;

#define DC_TRY(expr)                       \
    do {                                   \
        int _st = (expr);                  \
        if (_st != DC_B200_OK) return _st; \
    } while (0)

namespace {

// KS_APART: units from which on a launch of their own over all SMs pays its 4 us: a cluster of eight CTAs takes two rounds of loads for as many, and a step of 512 sequences with 64 K pages
// 226 us in one CTA, 21 in all SMs.
constexpr int KS_T = 1024, KS_PER = 4, KS_SLOTS = KS_T * KS_PER, KS_APART = 16 * KS_T;

struct StepParams {
    int slots, pages_per_seq, max_tokens, max_count;
    const int32_t *drop, *count;
    int32_t *lens, *held, *counts, *starts, *tables, *slot_map, *positions, *seqs, *drafts, *stack, *numbers;
    dc_kv_entry* entries;
    bool apart;                 // units are k_kv_places', which finds what it needs here:
    int32_t* scratch;
    struct Totals* totals;
};

// Exclusive sums of three values a thread over the CTA, in place; the whole sums to `all`.
struct Three {
    long long a;
    int b, c;
};
__device__ __forceinline__ void scan3(Three& x, Three* warps, Three& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Three in = x;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, in.a, s);
        const int b = __shfl_up_sync(0xffffffffu, in.b, s), c = __shfl_up_sync(0xffffffffu, in.c, s);
        if (lane >= s) in.a += a, in.b += b, in.c += c;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = in;
    __syncthreads();
    Three w = warps[lane], own = w;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, w.a, s);
        const int b = __shfl_up_sync(0xffffffffu, w.b, s), c = __shfl_up_sync(0xffffffffu, w.c, s);
        if (lane >= s) w.a += a, w.b += b, w.c += c;
    }
    all.a = __shfl_sync(0xffffffffu, w.a, 31), all.b = __shfl_sync(0xffffffffu, w.b, 31), all.c = __shfl_sync(0xffffffffu, w.c, 31);
    w.a -= own.a, w.b -= own.b, w.c -= own.c;
    x.a = in.a - x.a + __shfl_sync(0xffffffffu, w.a, warp), x.b = in.b - x.b + __shfl_sync(0xffffffffu, w.b, warp), x.c = in.c - x.c + __shfl_sync(0xffffffffu, w.c, warp);
}

// the last slot whose first number is at most x (first[0] = 0; slots without a number share the next one's first)
__device__ __forceinline__ int find(const int32_t* first, int n, int x) {
    int lo = 0, hi = n;      // first[lo] <= x < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Of every slot, ahead of it: new tokens, pages that they lie on, freed pages, granted ones; its tokens and pages that stay.
struct Slots {
    int32_t *tok0, *unit0, *free0, *give0, *keep, *left;
    __device__ __forceinline__ Slots(int32_t* at, int n) : tok0(at), unit0(at + n), free0(at + 2 * n), give0(at + 3 * n), keep(at + 4 * n), left(at + 5 * n) {}
};
enum { KS_ARRAYS = 6 };
struct Totals {
    int32_t tokens, units, freed, given, free;      // free: of the pool, before the step
};

// Units i .. i + 31, one a lane (a whole warp): pages that new tokens lie on, behind those freed ones that nobody takes.
__device__ __forceinline__ void place_units(const StepParams& p, const Slots& z, const Totals& all, int i) {
    const int lane = threadIdx.x & 31, n_units = all.units + max(0, all.freed - all.given);
    auto freed_page = [&](int j) {
        const int s = find(z.free0, p.slots, j);
        return p.tables[(size_t)s * p.pages_per_seq + z.left[s] + (j - z.free0[s])];
    };
    int s = 0, slot = 0, first = 0, t = 0, n = 0;
    i += lane;
    if (i < all.units) {
        s = find(z.unit0, p.slots, i);
        const int keep = z.keep[s], place = keep / DC_KV_BLOCK + i - z.unit0[s], tok0 = z.tok0[s], left = z.left[s];
        const int n_tok = (s + 1 < p.slots ? z.tok0[s + 1] : all.tokens) - tok0;
        int32_t* cell = p.tables + (size_t)s * p.pages_per_seq + place;
        int page;
        if (place < left) {
            page = *cell;
        } else {      // the j-th granted one
            const int j = z.give0[s] + place - left;
            page = j < all.freed ? freed_page(j) : p.stack[all.free - 1 - (j - all.freed)];
            *cell = page;
        }
        first = max(keep, place * DC_KV_BLOCK), n = min(keep + n_tok, (place + 1) * DC_KV_BLOCK) - first, t = tok0 + first - keep;
        slot = page * DC_KV_BLOCK + first % DC_KV_BLOCK;
    } else if (i < n_units) {
        const int j = all.given + i - all.units;
        p.stack[all.free + all.freed - 1 - j] = freed_page(j);
    }
    // ---- the units' tokens, two units at a time, a lane each
    const int x = lane & 15;
    for (uint32_t todo = __ballot_sync(0xffffffffu, n > 0); todo;) {
        const int a = __ffs(todo) - 1;
        todo &= todo - 1;
        const int b = todo ? __ffs(todo) - 1 : a, from = lane < 16 ? a : b;
        const bool mine = lane < 16 || todo != 0;
        todo &= todo - 1;
        const int us = __shfl_sync(0xffffffffu, s, from), uslot = __shfl_sync(0xffffffffu, slot, from), ufirst = __shfl_sync(0xffffffffu, first, from), ut = __shfl_sync(0xffffffffu, t, from),
                  un = __shfl_sync(0xffffffffu, n, from);
        if (mine && x < un) p.slot_map[ut + x] = uslot + x, p.positions[ut + x] = ufirst + x, p.seqs[ut + x] = us;
    }
}

__global__ void __launch_bounds__(KS_T) k_kv_step(const StepParams p) {
    extern __shared__ int32_t sm[];
    __shared__ Three warps[32];
    const Slots z(sm, p.slots);
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), n_cta = (int)cl.num_blocks();
    pdl_wait();
    pdl_launch_dependents();
    const int per = (p.slots + KS_T - 1) / KS_T, s0 = threadIdx.x * per;
    int left[KS_PER], kp[KS_PER], frees[KS_PER], cnt[KS_PER], asks[KS_PER];      // left: pages that stay
    Three x = {0, 0, 0}, all;
#pragma unroll
    for (int i = 0; i < KS_PER; ++i) {
        const int s = s0 + i;
        left[i] = kp[i] = frees[i] = cnt[i] = asks[i] = 0;
        if (i < per && s < p.slots) {
            const int len = p.lens[s], held = p.held[s];
            kp[i] = len - min(max(p.drop ? p.drop[s] : 0, 0), len);
            const int c = p.count ? p.count[s] : 0;
            cnt[i] = c >= 0 && c <= p.max_count && (long long)kp[i] + c <= (long long)p.pages_per_seq * DC_KV_BLOCK ? c : 0;
            const int need = (kp[i] + cnt[i] + DC_KV_BLOCK - 1) / DC_KV_BLOCK;
            left[i] = min(held, need), frees[i] = held - left[i], asks[i] = need - left[i];
            x.a += cnt[i], x.b += frees[i], x.c += asks[i];
        }
    }
    const int n_free = p.numbers[DC_KV_FREE];
    scan3(x, warps, all);
    const int n_freed = all.b;
    // ---- what is granted
    Three y = {0, 0, 0}, granted;      // a: new tokens and, 2^32 fold, pages that they lie on
    auto units = [&](int i) { return cnt[i] ? (kp[i] + cnt[i] - 1) / DC_KV_BLOCK - kp[i] / DC_KV_BLOCK + 1 : 0; };
    {
        long long tokens = x.a;
        int asked = x.c;
#pragma unroll
        for (int i = 0; i < KS_PER; ++i) {
            tokens += cnt[i], asked += asks[i];      // (at most the tables' places in all: below 2^31)
            if ((asks[i] && asked > n_free + n_freed) || tokens > p.max_tokens) cnt[i] = asks[i] = 0;
            y.a += cnt[i] + ((long long)units(i) << 32), y.b += asks[i], y.c += cnt[i] > 0;
        }
    }
    scan3(y, warps, granted);
    const Totals sum = {(int)granted.a, (int)(granted.a >> 32), n_freed, granted.b, n_free};
    {
        int tok = (int)y.a, unit = (int)(y.a >> 32), give = y.b, freed = x.b;
#pragma unroll
        for (int i = 0; i < KS_PER; ++i) {
            const int s = s0 + i;
            if (i >= per || s >= p.slots) break;
            z.tok0[s] = tok, z.unit0[s] = unit, z.give0[s] = give, z.free0[s] = freed, z.keep[s] = kp[i], z.left[s] = left[i];
            tok += cnt[i], unit += units(i), give += asks[i], freed += frees[i];
        }
    }
    if (n_cta > 1) cl.sync();      // everybody has read the old numbers
    else __syncthreads();
    if (rank == 0) {
        int entry = y.c;
        const Slots out(p.scratch, p.slots);
#pragma unroll
        for (int i = 0; i < KS_PER; ++i) {
            const int s = s0 + i;
            if (i >= per || s >= p.slots) break;
            p.lens[s] = kp[i] + cnt[i], p.held[s] = left[i] + asks[i], p.counts[s] = cnt[i], p.drafts[s] = cnt[i] - 1, p.starts[s] = z.tok0[s];
            if (cnt[i]) p.entries[entry++] = {s, kp[i], cnt[i], z.tok0[s]};
            if (p.apart) out.tok0[s] = z.tok0[s], out.unit0[s] = z.unit0[s], out.free0[s] = z.free0[s], out.give0[s] = z.give0[s], out.keep[s] = kp[i], out.left[s] = left[i];
        }
        if (threadIdx.x == 0) {
            p.starts[p.slots] = sum.tokens;
            p.numbers[DC_KV_FREE] = n_free + n_freed - sum.given;
            p.numbers[DC_KV_ENTRIES] = granted.c;
            if (p.apart) *p.totals = sum;
        }
    }
    if (p.apart) return;
    for (int i = rank * KS_T + (threadIdx.x & ~31); i < sum.units + max(0, n_freed - sum.given); i += n_cta * KS_T) place_units(p, z, sum, i);
}

// The units of a large step.
constexpr int KP_T = 512;
__global__ void __launch_bounds__(KP_T) k_kv_places(const StepParams p) {
    extern __shared__ int32_t sm[];
    pdl_wait();
    pdl_launch_dependents();
    const Totals sum = *p.totals;
    for (int i = threadIdx.x; i < KS_ARRAYS * p.slots; i += KP_T) sm[i] = p.scratch[i];
    __syncthreads();
    const Slots z(sm, p.slots);
    for (int i = blockIdx.x * KP_T + (threadIdx.x & ~31); i < sum.units + max(0, sum.freed - sum.given); i += gridDim.x * KP_T) place_units(p, z, sum, i);
}

__global__ void k_kv_stack(int32_t* stack, int n) {      // so that pages are handed out from 0 on
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) stack[i] = n - 1 - i;
}

// ---------------------------------------------------------------- new rows into the cache
struct WriteParams {
    const int32_t *starts, *counts, *slot_map, *seqs;
    int slots, max_tokens, n_kv, more_than;      // counts that are not more than this are left out
    const void *k, *v;
    int64_t ld;
    uint8_t* arena;
};

template <typename TC, typename TX>
__device__ __forceinline__ TC held_as(TX x);      // the cached form of a value
template <>
__device__ __forceinline__ __half held_as<__half, float>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __half held_as<__half, __half>(__half x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 held_as<__nv_bfloat16, __nv_bfloat16>(__nv_bfloat16 x) { return x; }

// A warp per (half of a run of new tokens within a page, key head); a lane has HD / 32 neighbouring dimensions.  Values are turned in registers: a dimension's tokens leave
// in sixteen-byte pieces where eight of them are new, one by one otherwise.
// Bound: latency of two rounds of loads, the tokens' places and the rows; a prompt's by its rows.
template <int HD, typename TX, typename TC>
__global__ void __launch_bounds__(128) k_kv16_write(const WriteParams p) {
    using R = dc_kv16_rec<HD>;
    constexpr int PER = HD / 32;
    struct alignas(PER * sizeof(TX)) Piece {
        TX x[PER];
    };
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, head = blockIdx.y, half = blockIdx.z, d0 = PER * lane;
    const bool vec = (((uintptr_t)p.k | (uintptr_t)p.v | (size_t)p.ld * sizeof(TX)) & (PER * sizeof(TX) - 1)) == 0;
    int T = 0x7fffffff;
    for (int t0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * DC_KV_BLOCK; t0 < T; t0 += gridDim.x * 4 * DC_KV_BLOCK) {
        // lane i: where token t0 + i lies, and whether it begins a run; the runs that begin with the first sixteen are the warp's
        const int t = min(t0 + lane, p.max_tokens - 1), slot = p.slot_map[t], seq = p.seqs[t], before = p.seqs[max(t - 1, 0)];
        T = p.starts[p.slots];
        const bool there = t0 + lane < T, begins = there && (slot % DC_KV_BLOCK == 0 || t == 0 || before != seq);
        const uint32_t all = __ballot_sync(0xffffffffu, begins), live = __ballot_sync(0xffffffffu, there);
        for (uint32_t todo = all & 0xFFFFu; todo; todo &= todo - 1) {
            const int from = __ffs(todo) - 1, tok = t0 + from, s = __shfl_sync(0xffffffffu, slot, from), at = s % DC_KV_BLOCK;
            const uint32_t behind = (all & ~((2u << from) - 1u)) | ~live;      // what ends the run
            const int n = (behind ? __ffs(behind) - 1 : 32) - from;
            const bool wanted = p.more_than == 0 || p.counts[__shfl_sync(0xffffffffu, seq, from)] > p.more_than;
            if (at >= 8 * half + 8 || at + n <= 8 * half) continue;
            const TX *k = reinterpret_cast<const TX*>(p.k) + (size_t)tok * p.ld + (size_t)head * HD + d0, *v = reinterpret_cast<const TX*>(p.v) + (size_t)tok * p.ld + (size_t)head * HD + d0;
            alignas(16) TX x[2][8][PER] = {};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * half + i - at;
                if (j < 0 || j >= n) continue;
                const TX *ks = k + (int64_t)j * p.ld, *vs = v + (int64_t)j * p.ld;
                if (vec) {
                    *reinterpret_cast<Piece*>(x[0][i]) = *reinterpret_cast<const Piece*>(ks);
                    *reinterpret_cast<Piece*>(x[1][i]) = *reinterpret_cast<const Piece*>(vs);
                } else {
#pragma unroll
                    for (int c = 0; c < PER; ++c) x[0][i][c] = ks[c], x[1][i][c] = vs[c];
                }
            }
            if (!wanted) continue;
            uint8_t* rec = p.arena + ((size_t)(s / DC_KV_BLOCK) * p.n_kv + head) * R::BYTES;
            alignas(16) TC kv[8][PER], vv[PER][8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < PER; ++c) kv[i][c] = held_as<TC, TX>(x[0][i][c]), vv[c][i] = held_as<TC, TX>(x[1][i][c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * half + i - at;
                if (j < 0 || j >= n) continue;
                uint8_t* to = rec + R::key(8 * half + i, d0);
                if constexpr (PER == 4) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(kv[i]);
                else *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(kv[i]);
            }
            if (at <= 8 * half && at + n >= 8 * half + 8) {
#pragma unroll
                for (int c = 0; c < PER; ++c) *reinterpret_cast<uint4*>(rec + R::value(8 * half, d0 + c)) = *reinterpret_cast<const uint4*>(vv[c]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int j = 8 * half + i - at;
                    if (j < 0 || j >= n) continue;
#pragma unroll
                    for (int c = 0; c < PER; ++c) *reinterpret_cast<TC*>(rec + R::value(8 * half + i, d0 + c)) = vv[c][i];
                }
            }
        }
    }
}

int check_call(dc_ctx* ctx, const dc_kv_cache* kv, const char* name) {
    if (!ctx || !kv) return DC_B200_INVALID_ARGUMENT;
    if (!kv->dev) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: not a cache whose sequences are on the GPU", name);
    if (kv->ctx != ctx) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: the cache belongs to another context", name);
    return DC_B200_OK;
}

int check_layer(dc_ctx* ctx, const dc_kv_cache* kv, int layer, const char* name) {
    DC_TRY(check_call(ctx, kv, name));
    if (layer < 0 || layer >= kv->dev->n_layer) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: layer %d of %d", name, layer, kv->dev->n_layer);
    if (kv->dev->max_count < 0) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "%s: no step yet (dc_b200_kv_step_dev)", name);
    return DC_B200_OK;
}

size_t element(int type) { return type == DC_TYPE_F32 ? 4 : 2; }

int create(dc_ctx* ctx, dc_kv_cache* kv) {
    dc_kv_dev& z = *kv->dev;
    kv->ctx = ctx;
    const size_t records = (size_t)z.pages * z.kv, bytes = records * 64 * z.dim * z.n_layer;
    z.layer_bytes = records * 64 * z.dim;
    const int ctas = dc_kv16_ctas(ctx->num_sms, z.kv);
    size_t at = 0;
    auto room = [&](size_t n) {
        const size_t from = at;
        at += (n + 255) / 256 * 256;
        return from;
    };
    const size_t slots4 = (size_t)z.slots * 4, tokens4 = (size_t)z.max_tokens * 4;
    const size_t lens = room(slots4), held = room(slots4), counts = room(slots4), starts = room(slots4 + 4), tables = room(slots4 * z.pages_per_seq), map = room(tokens4), positions = room(tokens4),
                 seqs = room(tokens4), drafts = room(slots4), numbers = room(DC_KV_NUMBERS * 4), entries = room(slots4 * 4), scratch = room(slots4 * KS_ARRAYS + sizeof(Totals)), tickets = room((size_t)ctas * z.kv * 4), stack = room((size_t)z.pages * 4), zeroed = at,
                 parts = room((size_t)2 * ctas * z.kv * dc_kv16_rows(z.type) * (z.dim + 2) * 4),
                 prompt_parts = room(z.type == DC_TYPE_F32 ? 0 : dc_kv16_prompt_parts(ctx->num_sms, z.kv, z.dim));
    DC_TRY(dc_check_cuda(ctx, cudaMalloc(&z.arena, bytes), "kv_create_dev"));
    DC_TRY(dc_check_cuda(ctx, cudaMalloc(&z.memory, at), "kv_create_dev"));
    DC_TRY(dc_check_cuda(ctx, cudaMemsetAsync(z.arena, 0, bytes, ctx->stream), "kv_create_dev"));
    DC_TRY(dc_check_cuda(ctx, cudaMemsetAsync(z.memory, 0, zeroed, ctx->stream), "kv_create_dev"));
    DC_TRY(dc_check_cuda(ctx, cudaMemsetAsync(z.memory + drafts, 0xFF, slots4, ctx->stream), "kv_create_dev"));
    auto ints = [&](size_t from) { return (int32_t*)(z.memory + from); };
    z.lens = ints(lens), z.held = ints(held), z.counts = ints(counts), z.starts = ints(starts), z.tables = ints(tables), z.slot_map = ints(map), z.positions = ints(positions), z.seqs = ints(seqs), z.drafts = ints(drafts);
    z.numbers = ints(numbers), z.entries = (dc_kv_entry*)(z.memory + entries), z.scratch = ints(scratch), z.tickets = ints(tickets), z.stack = ints(stack), z.parts = (float*)(z.memory + parts), z.prompt_parts = (float*)(z.memory + prompt_parts);
    DC_TRY(dc_launch_drained(ctx, "k_kv_stack", k_kv_stack, dim3(std::min((z.pages + 255) / 256, ctx->num_sms * 4)), dim3(256), 0, z.stack, z.pages));
    const int32_t free_pages = z.pages;
    DC_TRY(dc_check_cuda(ctx, cudaMemcpyAsync(z.numbers + DC_KV_FREE, &free_pages, 4, cudaMemcpyHostToDevice, ctx->stream), "kv_create_dev"));
    return dc_check_cuda(ctx, cudaStreamSynchronize(ctx->stream), "kv_create_dev");
}

template <int HD, typename TX, typename TC>
int launch_write(dc_ctx* ctx, const dc_kv_dev& z, const WriteParams& p) {
    const long long tokens = std::min<long long>(z.max_tokens, (long long)z.slots * z.max_count);
    const int ctas = (int)std::min<long long>((tokens + 4 * DC_KV_BLOCK - 1) / (4 * DC_KV_BLOCK), ctx->num_sms * 4);
    return dc_launch(ctx, "k_kv16_write", k_kv16_write<HD, TX, TC>, dim3(ctas, z.kv, 2), dim3(128), 0, p);
}

}  // namespace

int dc_launch_kv16_write(dc_ctx* ctx, const dc_kv_cache* kv, uint8_t* arena, const void* k, const void* v, int64_t ld, bool prompts_only) {
    const dc_kv_dev& z = *kv->dev;
    const WriteParams p = {z.starts, z.counts, z.slot_map, z.seqs, z.slots, z.max_tokens, z.kv, prompts_only ? dc_kv16_rows(z.type) / (z.heads / z.kv) : 0, k, v, ld, arena};
    if (z.dim == 128)
        return z.type == DC_TYPE_F32 ? launch_write<128, float, __half>(ctx, z, p)
               : z.type == DC_TYPE_F16 ? launch_write<128, __half, __half>(ctx, z, p) : launch_write<128, __nv_bfloat16, __nv_bfloat16>(ctx, z, p);
    return z.type == DC_TYPE_F32 ? launch_write<64, float, __half>(ctx, z, p)
           : z.type == DC_TYPE_F16 ? launch_write<64, __half, __half>(ctx, z, p) : launch_write<64, __nv_bfloat16, __nv_bfloat16>(ctx, z, p);
}

void dc_kv_dev_release(dc_kv_cache* kv) {
    dc_kv_dev* z = kv->dev;
    if (!z) return;
    if (z->arena) cudaFree(z->arena);
    if (z->memory) cudaFree(z->memory);
    delete z;
    kv->dev = nullptr;
}

extern "C" {

int dc_b200_kv_create_dev(dc_ctx* ctx, int n_layer, int n_head, int n_kv_head, int head_dim, int row_type, int max_blocks, int max_seqs, int max_blocks_per_seq, int max_tokens,
                          dc_kv_cache** out) {
    if (!ctx || !out) return DC_B200_INVALID_ARGUMENT;
    *out = nullptr;
    if (n_layer < 1 || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head || max_blocks < 1 || max_seqs < 1 || max_blocks_per_seq < 1 || max_tokens < 1)
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_create_dev: bad shape (%d heads, %d key heads)", n_head, n_kv_head);
    if (head_dim != 64 && head_dim != 128) return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_create_dev: head size %d (64 and 128 are supported)", head_dim);
    if (row_type != DC_TYPE_F32 && row_type != DC_TYPE_BF16 && row_type != DC_TYPE_F16)
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_create_dev: row type %d (F32, F16 and BF16 are supported)", row_type);
    if (max_seqs > KS_SLOTS || n_kv_head > 65535 || n_head > (1 << 20) || max_blocks > (1 << 26) || (long long)max_blocks_per_seq * DC_KV_BLOCK > (1 << 30) ||
        (long long)max_seqs * max_blocks_per_seq > (1LL << 31) - 1 || (long long)max_tokens * n_head > (1 << 30) || (long long)n_layer * max_blocks * n_kv_head > (1LL << 40))
        return dc_fail(ctx, DC_B200_UNSUPPORTED, "kv_create_dev: %d sequences of %d pages, %d pages, %d heads, %d new tokens", max_seqs, max_blocks_per_seq, max_blocks, n_head, max_tokens);
    cudaSetDevice(ctx->device);
    dc_kv_cache* kv = nullptr;
    int st;
    try {
        kv = new dc_kv_cache();
        kv->dev = new dc_kv_dev();
        dc_kv_dev& z = *kv->dev;
        z.n_layer = n_layer, z.heads = n_head, z.kv = n_kv_head, z.dim = head_dim, z.type = row_type, z.slots = max_seqs, z.pages = max_blocks, z.pages_per_seq = max_blocks_per_seq;
        z.max_tokens = max_tokens;
        st = create(ctx, kv);
    } catch (const std::bad_alloc&) {
        st = dc_fail(ctx, DC_B200_OUT_OF_MEMORY, "kv_create_dev: out of host memory");
    }
    if (st != DC_B200_OK && kv) {
        dc_kv_release(kv);
        delete kv;
        kv = nullptr;
    }
    *out = kv;
    return st;
}

int dc_b200_kv_dev_arrays(dc_kv_cache* kv, dc_kv_dev_arrays* out) {
    if (!kv || !out) return DC_B200_INVALID_ARGUMENT;
    if (!kv->dev) return dc_fail(kv->ctx, DC_B200_INVALID_ARGUMENT, "kv_dev_arrays: not a cache whose sequences are on the GPU");
    const dc_kv_dev& z = *kv->dev;
    *out = {z.lens, z.counts, z.starts, z.tables, z.slot_map, z.positions, z.seqs, z.numbers + DC_KV_FREE};
    return DC_B200_OK;
}

int dc_b200_kv_dev_drafts(dc_kv_cache* kv, const int32_t** drafts_dev_out) {
    if (!kv || !drafts_dev_out) return DC_B200_INVALID_ARGUMENT;
    if (!kv->dev) return dc_fail(kv->ctx, DC_B200_INVALID_ARGUMENT, "kv_dev_drafts: not a cache whose sequences are on the GPU");
    *drafts_dev_out = kv->dev->drafts;
    return DC_B200_OK;
}

int dc_b200_kv_step_dev(dc_ctx* ctx, dc_kv_cache* kv, const int32_t* drop_dev, const int32_t* count_dev, int max_count) {
    DC_TRY(check_call(ctx, kv, "kv_step_dev"));
    dc_kv_dev& z = *kv->dev;
    if (max_count < 0) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_step_dev: at most %d new tokens a sequence", max_count);
    if (((uintptr_t)drop_dev | (uintptr_t)count_dev) % 4) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_step_dev: an array is not aligned to its elements");
    cudaSetDevice(ctx->device);
    // pages that new tokens may lie on, and that may be freed: a CTA of 1024 threads, a cluster of eight, or all SMs behind a launch of their own
    const long long units = (long long)z.slots * std::min<long long>(max_count / DC_KV_BLOCK + 2, z.pages_per_seq);
    const bool apart = units > KS_APART;
    const StepParams p = {z.slots, z.pages_per_seq, z.max_tokens, max_count, drop_dev, count_dev, z.lens, z.held, z.counts, z.starts, z.tables, z.slot_map, z.positions, z.seqs, z.drafts, z.stack,
                          z.numbers, z.entries, apart, z.scratch, (Totals*)(z.scratch + (size_t)KS_ARRAYS * z.slots)};
    const size_t smem = (size_t)z.slots * KS_ARRAYS * 4;
    DC_TRY(dc_kernel_setup(ctx, (const void*)k_kv_step, KS_SLOTS * KS_ARRAYS * 4, "k_kv_step"));
    const int n_cta = !apart && (units > 4 * KS_T || (drop_dev && (long long)z.slots * z.pages_per_seq > 64 * KS_T)) ? 8 : 1;
    DC_TRY(dc_launch_cluster(ctx, "k_kv_step", k_kv_step, dim3(n_cta), dim3(KS_T), smem, n_cta, p));
    if (apart) {
        DC_TRY(dc_kernel_setup(ctx, (const void*)k_kv_places, KS_SLOTS * KS_ARRAYS * 4, "k_kv_places"));
        DC_TRY(dc_launch(ctx, "k_kv_places", k_kv_places, dim3((unsigned)std::min<long long>((units + KP_T - 1) / KP_T, 2 * ctx->num_sms)), dim3(KP_T), smem, p));
    }
    z.max_count = max_count;
    return DC_B200_OK;
}

int dc_b200_kv_dev_write_dev(dc_ctx* ctx, dc_kv_cache* kv, int layer, const void* k_dev, const void* v_dev, int64_t ld_kv) {
    DC_TRY(check_layer(ctx, kv, layer, "kv_dev_write_dev"));
    const dc_kv_dev& z = *kv->dev;
    if (ld_kv == 0) ld_kv = (int64_t)z.kv * z.dim;
    if (!k_dev || !v_dev || ld_kv < (int64_t)z.kv * z.dim || ((uintptr_t)k_dev | (uintptr_t)v_dev) % element(z.type))
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "kv_dev_write_dev: bad argument (row stride %lld)", (long long)ld_kv);
    if (z.max_count == 0) return DC_B200_OK;
    cudaSetDevice(ctx->device);
    return dc_launch_kv16_write(ctx, kv, z.arena + z.layer_bytes * layer, k_dev, v_dev, ld_kv, false);
}

int dc_b200_flash_attn_kv_dev(dc_ctx* ctx, dc_kv_cache* kv, int layer, const void* q_dev, int64_t ld_q, const void* k_dev, const void* v_dev, int64_t ld_kv, float scale, int window,
                              int keep_first, void* out_dev, int64_t ld_out) {
    DC_TRY(check_layer(ctx, kv, layer, "flash_attn_kv_dev"));
    const dc_kv_dev& z = *kv->dev;
    const int64_t q_row = (int64_t)z.heads * z.dim, kv_row = (int64_t)z.kv * z.dim;
    if (ld_q == 0) ld_q = q_row;
    if (ld_kv == 0) ld_kv = kv_row;
    if (ld_out == 0) ld_out = q_row;
    if (!q_dev || !out_dev || (!k_dev != !v_dev) || ld_q < q_row || ld_out < q_row || ld_kv < kv_row ||
        ((uintptr_t)q_dev | (uintptr_t)k_dev | (uintptr_t)v_dev | (uintptr_t)out_dev) % element(z.type))
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "flash_attn_kv_dev: bad argument (row strides %lld, %lld, %lld)", (long long)ld_q, (long long)ld_kv, (long long)ld_out);
    if (!isfinite(scale)) return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "flash_attn_kv_dev: scale is not finite");
    if (window < 0 || keep_first < 0 || (keep_first > 0 && window == 0))
        return dc_fail(ctx, DC_B200_INVALID_ARGUMENT, "flash_attn_kv_dev: window %d, first tokens kept %d", window, keep_first);
    if (z.max_count == 0) return DC_B200_OK;
    cudaSetDevice(ctx->device);
    const dc_kv16_call c = {kv, z.arena + z.layer_bytes * layer, q_dev, k_dev, v_dev, ld_q, ld_kv, ld_out, scale, window, keep_first, out_dev};
    if ((long long)z.max_count * (z.heads / z.kv) > dc_kv16_rows(z.type)) {      // sequences with more rows than a CTA takes: their rows are written ahead of all
        if (k_dev) DC_TRY(dc_launch_kv16_write(ctx, kv, c.arena, k_dev, v_dev, ld_kv, true));
        DC_TRY(z.type == DC_TYPE_F32 ? dc_launch_kv16_rows(ctx, c, true) : dc_launch_kv16_prompt(ctx, c));
    }
    return dc_launch_kv16_rows(ctx, c, false);
}

int dc_b200_kv_dev_read_page(dc_kv_cache* kv, int layer, int block, void* k_host, void* v_host) {
    if (!kv || !kv->dev || layer < 0 || layer >= kv->dev->n_layer || block < 0 || block >= kv->dev->pages) return DC_B200_INVALID_ARGUMENT;
    const dc_kv_dev& z = *kv->dev;
    cudaSetDevice(kv->ctx->device);
    const size_t page = (size_t)64 * z.dim * z.kv;
    uint8_t* from = new (std::nothrow) uint8_t[page];
    if (!from) return dc_fail(kv->ctx, DC_B200_OUT_OF_MEMORY, "kv_dev_read_page: out of host memory");
    cudaError_t e = cudaStreamSynchronize(kv->ctx->stream);
    if (e == cudaSuccess) e = cudaMemcpy(from, z.arena + z.layer_bytes * layer + page * block, page, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess)
        for (int tok = 0; tok < DC_KV_BLOCK; ++tok)
            for (int h = 0; h < z.kv; ++h)
                for (int d = 0; d < z.dim; ++d) {
                    const uint8_t* r = from + (size_t)h * 64 * z.dim;
                    const size_t to = (((size_t)tok * z.kv + h) * z.dim + d) * 2;
                    if (k_host) memcpy((uint8_t*)k_host + to, r + (z.dim == 128 ? dc_kv16_rec<128>::key(tok, d) : dc_kv16_rec<64>::key(tok, d)), 2);
                    if (v_host) memcpy((uint8_t*)v_host + to, r + (z.dim == 128 ? dc_kv16_rec<128>::value(tok, d) : dc_kv16_rec<64>::value(tok, d)), 2);
                }
    delete[] from;
    return dc_check_cuda(kv->ctx, e, "kv_dev_read_page");
}

}  // extern "C"
