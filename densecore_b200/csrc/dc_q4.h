// A cache of keys and values in 4 bits: where everything lies, and the plan of a step.  Shared by attn_q4.cu and attn_q4_prompt.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

#include "dc_kv.h"

// A page of a key head is one record of 18 HD bytes, so that one bulk copy brings it:
//   key codes     8 HD   words of eight codes of one token, in the order in which lanes of mma.m16n8k16 take a second operand of 16 dimensions x 8 tokens
//   key scales      HD   [16 tokens][HD / 64] pairs (scale, least value) of fp16
//   value codes   8 HD   the same for 16 tokens x 8 dimensions; a byte is two dimensions (d, d + 8) of one token
//   value scales    HD
// Every byte belongs to one token: tokens are written one by one, by different warps, without reading what is there.
template <int HD>
struct dc_q4_rec {
    static constexpr int GROUPS = HD / 64, K_SCALES = 8 * HD, V_CODES = 9 * HD, V_SCALES = 17 * HD, BYTES = 18 * HD;
    // word i (dimensions 32 i ..) of lane t's part of a token's key: nibble q + 4 o holds dimension 32 i + 8 q + 2 t + o
    static constexpr int __host__ __device__ k_word(int tok, int t, int i) {
        return HD == 128 ? (tok >> 3) * 512 + ((tok & 7) * 4 + t) * 16 + 4 * i : ((tok & 7) * 4 + t) * 16 + (tok >> 3) * 8 + 4 * i;
    }
    // byte of dimensions 16 i + d8 (low nibble) and 16 i + 8 + d8 (high nibble) of a token's value
    static constexpr int __host__ __device__ v_byte(int tok, int d8, int i) {
        const int lane = d8 * 4 + ((tok & 7) >> 1);
        return V_CODES + (HD == 128 ? (i >> 2) * 512 + lane * 16 + (i & 3) * 4 : lane * 16 + i * 4) + (tok >> 3) + 2 * (tok & 1);
    }
};

// The plan of a step in device memory: arrays in one allocation, which a larger plan replaces, and this header, which stays where it is as long as the cache does.
// Kernels get the arrays' places from the host and read the counts, so that they need not wait for one to find the other; within a captured call they take the
// places from the header, so that it serves every later plan, wherever that lies.
struct dc_q4_token {
    int32_t block, slot;
};
struct dc_q4_item;
struct dc_q4_head {
    int32_t T, n_items, n_tiles, n_joins;
    const dc_q4_token* tokens;
    const dc_q4_item* items;
    int32_t* tickets;
    float* ws;
};
// One CTA's work in k_q4_rows: pages page0 .. page1 - 1 for one tile of eight rows (row r: new token r / G of the entry, query head r % G of the key head).
struct dc_q4_item {
    int32_t seq, pos0, tok0, count, tile, page0, page1;
    int32_t split, n_splits, ws;      // of the tile; partial results at ws + split
    int32_t ticket, pad;
};
// One CTA's work in k_q4_prompt: up to 256 rows from row0 of the entry on, key tiles (64 keys) tile0 .. tile1 - 1 of the ones that they see; partial results at ws + split.
struct dc_q4_tile {
    int32_t seq, pos0, tok0, count, row0, tile0, tile1, split, n_splits, ws, pad[2];
};

// `count` new tokens of a sequence from position pos0 on; the step's tokens tok0 ..
struct dc_q4_entry {
    int32_t seq, pos0, count, tok0;
};
constexpr int DC_Q4_WARPS = 4;      // of a CTA of k_q4_rows
constexpr int DC_Q4_SPLITS = 240;   // of a tile, at most

// The items of all tiles of the entries; *n_ws: partial results, *n_tickets: tiles that more than one CTA works on.
inline void dc_q4_items(const std::vector<dc_q4_entry>& es, int G, int n_kv, int num_sms, std::vector<dc_q4_item>* items, int* n_tickets, int* n_ws) {
    auto tiles_of = [&](const dc_q4_entry& e) { return (int)(((long long)e.count * G + 7) / 8); };
    auto pages_of = [&](const dc_q4_entry& e, int tile) { return (e.pos0 + std::min(e.count - 1, (tile * 8 + 7) / G)) / 16 + 1; };
    long long work = 0;
    for (const dc_q4_entry& e : es)
        for (int t = 0; t < tiles_of(e); ++t) work += pages_of(e, t);
    // pages of an item: about three rounds of the four CTAs that an SM holds (bf16 rows; three: f32) where there is that much, six pages a warp at least (joining parts takes as long as some five
    // pages).  48 requests of up to 32000 positions: 179 us with a third of the items, 163 with two thirds, 162, 164 with four thirds, 185 with eight
    const long long slots = (long long)num_sms * 3 * 4;
    const int per = (int)std::max<long long>(6 * DC_Q4_WARPS, (work * n_kv + slots - 1) / slots);
    *n_tickets = *n_ws = 0;
    for (const dc_q4_entry& e : es)
        for (int t = 0; t < tiles_of(e); ++t) {
            const int pages = pages_of(e, t), mine = std::max(per, (pages + DC_Q4_SPLITS - 1) / DC_Q4_SPLITS), n = (pages + mine - 1) / mine;
            for (int s = 0; s < n; ++s)
                items->push_back({e.seq, e.pos0, e.tok0, e.count, t, s * mine, std::min(pages, (s + 1) * mine), s, n, n > 1 ? *n_ws : 0, n > 1 ? *n_tickets : 0, 0});
            if (n > 1) ++*n_tickets, *n_ws += n;
        }
}

// Entries of that many rows (new tokens times query heads of a key head) take the tensor-core kernel, for bf16 rows.
constexpr int DC_Q4_PROMPT_ROWS = 64;

// Tiles of the entries for k_q4_prompt, those with most keys first.  Keys are split where there are fewer tiles than SMs, into parts of eight key tiles at least.
inline void dc_q4_tiles(const std::vector<dc_q4_entry>& es, int G, int n_kv, int num_sms, std::vector<dc_q4_tile>* tiles, int* n_ws) {
    *n_ws = 0;
    long long n = 0;
    for (const dc_q4_entry& e : es) n += ((long long)e.count * G + 255) / 256;
    const int most = n ? (int)std::max<long long>(1, num_sms / (n * n_kv)) : 1;
    for (const dc_q4_entry& e : es)
        for (int r = 0; r < e.count * G; r += 256) {
            const int keys = (e.pos0 + (std::min(r + 256, e.count * G) - 1) / G) / 64 + 1, parts = std::max(1, std::min(most, keys / 8));
            for (int s = 0; s < parts; ++s)
                tiles->push_back({e.seq, e.pos0, e.tok0, e.count, r, (int)((long long)keys * s / parts), (int)((long long)keys * (s + 1) / parts), s, parts, parts > 1 ? *n_ws : 0, {0, 0}});
            if (parts > 1) *n_ws += parts;
        }
    std::stable_sort(tiles->begin(), tiles->end(), [](const dc_q4_tile& a, const dc_q4_tile& b) { return a.tile1 - a.tile0 > b.tile1 - b.tile0; });
}

struct dc_q4 {
    int n_layer = 0, heads = 0, kv = 0, dim = 0, type = 0;
    // the newest plan: host copies of what launches need, and the block manager's state that it was made for
    bool planned = false;
    uint64_t edits = 0;
    int T = 0, n_items = 0, n_tiles = 0, n_joins = 0;
    dc_q4_head* head = nullptr;         // device
    uint8_t* plan = nullptr;            // arrays
    size_t cap[7] = {}, at[7] = {};     // room for the arrays and where they begin: tokens, items, tiles, joins, tickets, partial results of rows and of prompt tiles
    std::vector<uint8_t*> retired;      // outgrown plans, which calls in flight may still read
    uint8_t* stage = nullptr;           // pinned copy of the plan being uploaded
    size_t stage_bytes = 0;
    cudaEvent_t uploaded = nullptr;
};

enum { DC_Q4_TOKENS = 0, DC_Q4_ITEMS, DC_Q4_TILES, DC_Q4_JOINS, DC_Q4_TICKETS, DC_Q4_WS, DC_Q4_PARTS, DC_Q4_ARRAYS };

struct dc_q4_call {
    const dc_kv_cache* kv;
    const uint8_t* arena;      // one layer
    const void* q;
    int ldq, ldo;
    float scale;
    void* out;
    int early;                 // what k_q4_rows may do ahead of its predecessor's end: 0 nothing, 1 all but the step's own pages and stores (k_q4_write), 2 everything
                               // (k_q4_prompt of the same call, whose CTAs have begun, behind k_q4_write)
    bool captured;             // the call is being captured: its replays take the newest plan from the header
};
int dc_launch_q4_rows(dc_ctx* ctx, const dc_q4_call& c);
int dc_launch_q4_prompt(dc_ctx* ctx, const dc_q4_call& c);
int dc_launch_q4_join(dc_ctx* ctx, const dc_q4_call& c);      // last: adds up the prompt tiles whose keys are split
