// Row tiles of prompt-sized sequences, as the kernel that works on them and the one that adds up their parts find them.
#pragma once
#include "dc_common.cuh"
#include "dc_kv_dev.h"

namespace dc {

constexpr int KP_ROWS = 128, KP_TILE_ROWS = 2 * KP_ROWS;      // rows of a set, of a tile
template <int HD>
constexpr int kp_part_floats() { return KP_TILE_ROWS * (HD + 4); }      // of a part: rows of HD answers, the reference and the sum of their weights

// Pages that tokens at positions `first` .. `last` see, numbered: the first `kept` ones, then those from `low` on.
struct Pages {
    int kept, low, n;
    __device__ __forceinline__ int at(int i) const { return i < kept ? i : low + i - kept; }
};
__device__ __forceinline__ Pages pages_of(int first, int last, int window, int keep) {
    Pages g;
    g.low = window ? max(0, first - window + 1) / DC_KV_BLOCK : 0;
    g.kept = min((int)(((long long)keep + DC_KV_BLOCK - 1) / DC_KV_BLOCK), g.low);
    g.n = g.kept + last / DC_KV_BLOCK - g.low + 1;
    return g;
}

// The tiles of all sequences with more than `least` rows stand in a line.  Found by whole warps.
struct TileLine {
    const dc_kv_entry* entries;
    int n_entries, G, least, n_all, most;      // n_all: tiles; most: parts of a tile's keys at most, where there are fewer tiles than SMs
    __device__ __forceinline__ int tiles_of(const dc_kv_entry& e) const {
        const int rows = e.count * G;      // (at most 2^30, as the whole step's)
        return rows > least ? (rows + KP_TILE_ROWS - 1) / KP_TILE_ROWS : 0;
    }
    dc_kv_entry early;      // the lane's of the first 32, on its way with their number
    __device__ __forceinline__ dc_kv_entry entry(int base) const {
        const int i = base + (threadIdx.x & 31);
        return i >= n_entries ? dc_kv_entry{0, 0, 0, 0} : base == 0 ? early : entries[i];
    }
    // slots: room for entries
    __device__ __forceinline__ TileLine(const dc_kv_entry* e, const int32_t* n, int slots, int G_, int least_, int n_kv, int num_sms) : entries(e), G(G_), least(least_), n_all(0) {
        early = e[min((int)(threadIdx.x & 31), slots - 1)];
        n_entries = *n;
        for (int base = 0; base < n_entries; base += 32) n_all += tiles_of(entry(base));
        n_all = __reduce_add_sync(0xffffffffu, n_all);
        most = n_all ? max(1, num_sms / (int)min((long long)n_all * n_kv, (long long)num_sms)) : 1;
    }
};
struct Tile {
    dc_kv_entry e;
    int row0, rows, first, last;      // rows from row0 on, the positions of the first and the last one's tokens
    Pages pages;
    int key_tiles, n_parts;
    // tile i of the line, i < n_all
    __device__ __forceinline__ Tile(const TileLine& z, int i, int window, int keep) {
        const int lane = threadIdx.x & 31;
        int before = 0, tile = 0;
        for (int base = 0;; base += 32) {
            e = z.entry(base);
            const int mine = z.tiles_of(e);
            int upto = mine;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, upto, s);
                if (lane >= s) upto += o;
            }
            const uint32_t there = __ballot_sync(0xffffffffu, before + upto > i);
            if (there) {
                const int who = __ffs(there) - 1;
                tile = __shfl_sync(0xffffffffu, before + upto, who) - 1 - i;      // the last tile first: it sees most keys
                e.seq = __shfl_sync(0xffffffffu, e.seq, who), e.pos0 = __shfl_sync(0xffffffffu, e.pos0, who);
                e.count = __shfl_sync(0xffffffffu, e.count, who), e.tok0 = __shfl_sync(0xffffffffu, e.tok0, who);
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        row0 = tile * KP_TILE_ROWS, rows = min(KP_TILE_ROWS, e.count * z.G - row0);
        first = e.pos0 + row0 / z.G, last = e.pos0 + (row0 + rows - 1) / z.G;
        pages = pages_of(first, last, window, keep);
        key_tiles = (pages.n + 3) / 4, n_parts = max(1, min(z.most, key_tiles / 8));
    }
};

}  // namespace dc
