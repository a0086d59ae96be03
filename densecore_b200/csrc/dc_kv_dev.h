// A paged cache of 16-bit rows whose sequences are kept on the GPU: where everything lies.  Shared by kv_dev.cu, attn_kv16.cu and attn_kv16_prompt.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "dc_kv.h"

// A page of a key head is one record of 64 HD bytes, so that one bulk copy brings it, laid out as matrix instructions take it:
//   keys     32 HD   groups of eight tokens, of 64 dimensions each time: rows of 128 bytes, one token's, chunk c (16 bytes) of row r at place c ^ (r & 7): the 128-byte
//                    swizzle of tcgen05 operands, whose 8-row groups are 16 HD bytes apart over all pages of a tile; ldmatrix meets no bank twice
//   values   32 HD   turned: rows of 32 bytes are dimensions, the sixteen tokens along them, chunk c of row r at place c ^ (r >> 2 & 1): the 32-byte swizzle
template <int HD>
struct dc_kv16_rec {
    static constexpr uint32_t VALUES = 32 * HD, BYTES = 64 * HD, GROUP = 16 * HD;
    static constexpr uint32_t __host__ __device__ key(int tok, int d) {
        return (tok >> 3) * GROUP + (d >> 6) * 1024 + (tok & 7) * 128 + ((((d >> 3) & 7) ^ (tok & 7)) << 4) + (d & 7) * 2;
    }
    static constexpr uint32_t __host__ __device__ value(int tok, int d) { return VALUES + d * 32 + (((tok >> 3) ^ ((d >> 2) & 1)) << 4) + (tok & 7) * 2; }
};

// A sequence with new tokens in the step: its slot, its tokens before them, their number, the step's tokens ahead of them.
struct alignas(16) dc_kv_entry {
    int32_t seq, pos0, count, tok0;
};

// Device arrays; they stay where they are as long as the cache does.
struct dc_kv_dev {
    int n_layer = 0, heads = 0, kv = 0, dim = 0, type = 0, slots = 0, pages = 0, pages_per_seq = 0, max_tokens = 0;
    int max_count = -1;            // of the newest step; -1: none yet
    size_t layer_bytes = 0;
    uint8_t* arena = nullptr;      // [layer][page][key head] records
    int32_t *lens = nullptr, *held = nullptr, *counts = nullptr, *starts = nullptr, *tables = nullptr, *slot_map = nullptr, *positions = nullptr, *seqs = nullptr, *drafts = nullptr, *stack = nullptr;
    int32_t* numbers = nullptr;    // free pages, entries
    int32_t* scratch = nullptr;    // of a step
    dc_kv_entry* entries = nullptr;
    uint8_t* memory = nullptr;     // all of the above but the arena
    // of attention: partial results and tickets of sequences that several CTAs work on (zero between calls)
    float *parts = nullptr, *prompt_parts = nullptr;
    int32_t* tickets = nullptr;
};
enum { DC_KV_FREE = 0, DC_KV_ENTRIES = 1, DC_KV_NUMBERS = 4 };

// Rows (new tokens times query heads of a key head) of a sequence that one CTA of the rows kernel takes at a time; sequences with more are prompt-sized.
inline int dc_kv16_rows(int type) { return type == 0 ? 32 : 64; }
// CTAs a key head of the rows kernel: three an SM
inline int dc_kv16_ctas(int num_sms, int n_kv) { const int n = 3 * num_sms / n_kv; return n < 1 ? 1 : n; }

struct dc_kv16_call {
    const dc_kv_cache* kv;
    uint8_t* arena;                // of the layer
    const void *q, *k, *v;         // k, v null: the rows stand in the cache
    int64_t ldq, ldkv, ldo;
    float scale;
    int window, keep;
    void* out;
};
int dc_launch_kv16_write(dc_ctx* ctx, const dc_kv_cache* kv, uint8_t* arena, const void* k, const void* v, int64_t ld, bool prompts_only);
int dc_launch_kv16_rows(dc_ctx* ctx, const dc_kv16_call& c, bool prompts);
int dc_launch_kv16_prompt(dc_ctx* ctx, const dc_kv16_call& c);      // prompt-sized sequences of 16-bit rows
size_t dc_kv16_prompt_parts(int num_sms, int n_kv, int dim);        // bytes of its partial results
