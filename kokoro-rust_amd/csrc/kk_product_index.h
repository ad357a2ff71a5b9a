// kk_product_index.h -- which tiles the blocks of the products take, and how a product is launched: plain index arithmetic, the same
// functions on the host (tests/product_index_check.hip walks every block of random launches with them) and in the kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kk_common.h"
#include "kk_kv_index.h"
#include "kokoro_hip.h"

namespace kk {

// Rows `first`..`first + count` (count <= M) of group g.
struct Rows {
    int g, first, count;
};

// Row tiles of a group: as many as its rows need.  A tile's number counts those of the groups before it.
__host__ __device__ inline int64_t row_tiles(int64_t entries, int groups, int M) {  // at most
    const int64_t n = entries / M + groups;
    return n < entries ? n : entries;
}
__host__ __device__ inline bool group_ok(int s0, int s1, int entries) { return s0 >= 0 && s1 >= s0 && s1 <= entries; }
// Tile i of group g, whose rows are [s0, s1).
__host__ __device__ inline void group_rows(int s0, int s1, int g, int i, int M, Rows& r) {
    r.g = g, r.first = s0 + i * M;
    const int left = s1 - r.first;
    r.count = left < M ? left : M;
}

// The tiles that block `block` of `blocks` (a multiple of 8) takes of `total`: from `first` on, every blocks / 8, below `end`.  Blocks go to the
// 8 XCDs in turn; an XCD takes tiles that follow each other, which share rows of x and matrices in its L2.
struct TileWalk {
    int first, step, end;
};
__host__ __device__ inline TileWalk tile_walk(int block, int blocks, int total) {
    const int per = (total + 7) / 8, stop = (block % 8 + 1) * per;
    return {block % 8 * per + block / 8, blocks / 8, stop < total ? stop : total};
}
// Tile t of `tall` rows of tiles, each tiles_n wide: strips eight tiles of outputs wide, so that the 32 CUs of an XCD share 4 x 8 tiles.
struct TileAt {
    int n, row;
};
__host__ __device__ inline TileAt tile_at(int t, int tall, int tiles_n) {
    const int strip = t / (8 * tall), left = tiles_n - 8 * strip, wide = left < 8 ? left : 8, in = t - strip * (8 * tall), row = in / wide;
    return {8 * strip + (in - row * wide), row};
}

// ------------------------------------------------------------------ host side

// How a product is launched.
enum { k64, k128, k128Wide, k256 };  // tiles, by their rows of x
struct ProductPlan {
    int tile;
    int blocks, tiles, tiles_n, splits, k_split;
    int64_t shrink;  // blocks of the adapters' h
};
struct AdapterPlan {
    ProductPlan main, rest;  // of the first `rows` rows and of those behind
    int rows;
    bool joined;     // parts of the main product are summed, and the adapters' share added, by a kernel of their own
    int slots, h_splits, h_k;
    int64_t ws_h2, ws_unit, ws_part, ws_bytes;  // workspace
};
inline bool product_fits(const ProductPlan& p) {
    return p.shrink * 512 <= kMostThreads / 2 && (int64_t)p.tiles * p.tiles_n * p.splits <= 1 << 27;
}

struct TileSize {
    int N, M, per_cu;
};
constexpr TileSize kTiles[] = {{128, 64, 2}, {64, 128, 2}, {256, 128, 1}, {256, 256, 1}};

// The grid: as many blocks as tiles or as the device holds at once.
inline void size_grid(ProductPlan& p, int64_t row_tiles, int64_t wide, int n_cu) {
    const TileSize& z = kTiles[p.tile];
    p.tiles = (int)row_tiles, p.tiles_n = (int)ceil_div(wide, z.N);
    const int64_t all = row_tiles * p.tiles_n * p.splits;
    p.blocks = (int)((std::min<int64_t>(all, (int64_t)z.per_cu * n_cu) + 7) / 8 * 8);
}

inline ProductPlan expert_plan(const kk_expert_product_args& a, int n_cu) {
    ProductPlan p{};
    p.splits = 1, p.k_split = a.inputs;
    const int64_t mean = a.entries / a.groups;
    // Measured, us, tiles of 64, 128 and 256 rows: 64 groups of 1,024 x 2,048 with 8 rows each 50, 51, 57; 32: 57, 57, 63; 62: 64, 70, 70;
    // 125: 88, 79, 104; 250: 146, 113, 118; 500: 273, 210, 199.  (Tiles of 32 rows: 53, 64, 88.)
    const int64_t wide = (int64_t)a.outputs * (a.gate != KK_GATE_NONE ? 2 : 1);
    auto tiles = [&](int tile) { return a.groups * ceil_div(mean, kTiles[tile].M) * ceil_div(wide, kTiles[tile].N); };
    // Where the device holds all tiles of 64 rows at once, they leave the fewest CUs idle: 8 groups of 2 x 1,024 x 2,048 with 60 rows each 16
    // us (of 128 rows 27), 150: 23 (27), 200: 24 (28); 16 groups with 100: 45 (44).  Tiles of 256 rows where their rounds are full: 8 groups
    // of 4,096 x 4,096 with 900 rows (2 rounds) 267 (of 128 rows 281), with 600 (1.5) 230 (202); 16 of 2 x 1,024 x 2,048 131 (140), 116 (105).
    const int64_t large = tiles(k256), room = ceil_div(large, n_cu) * n_cu;
    p.tile = mean <= 40 || tiles(k64) <= 2 * n_cu ? k64 : mean < 450 || large * 10 < room * 9 ? k128Wide : k256;
    size_grid(p, row_tiles(a.entries, a.groups, kTiles[p.tile].M), wide, n_cu);
    return p;
}

inline AdapterPlan adapter_plan(const kk_adapter_product_args& a, int n_cu) {
    AdapterPlan r{};
    ProductPlan& p = r.main;
    p.splits = 1, p.k_split = a.inputs;
    auto tiles = [&](int64_t rows, int tile) { return ceil_div(rows, kTiles[tile].M) * ceil_div(a.outputs, kTiles[tile].N); };
    // us here and below, of 4,096 inputs and outputs where no other are named, both sides measured.  Tiles of 128 rows where they take three
    // quarters of the CUs: 1,024 rows (half of the CUs) 56, with tiles of 64 51; 1,280 61, 74 (with ten adapters of rank 32 75, 83); 1,600 59, 85;
    // 1,900 65, 96.
    p.tile = tiles(a.rows, k128Wide) * 4 >= 3 * n_cu ? k128Wide : k64;
    // Parts only where even the smaller tiles leave CUs idle: 1,500 rows of 4,096 x 4,096 69 us without, 111 with them
    r.joined = tiles(a.rows, k64) < n_cu;
    int64_t rows = a.rows;
    if (r.joined) {
        // tiles of 64 rows and of 128, 6,144 outputs: 32 rows 17, 21; 64: 20, 23; 96: 25.6, 25.4; 128: 27.4, 27.3; 256 rows 26.6, 27.0
        p.tile = a.rows <= 64 ? k64 : k128;
        // A block for each CU where that splits the inputs, else two: 96 tiles in 2 parts take as long as in 5, with less to sum up.  Parts of 512
        // inputs or more (of 256, of 1,024): one row 12.1 (12.0, 13.2); 16 rows of 2,048 x 1,024 9.1 (8.5, 10.5); 64 rows of 768 x 768 11.2 (9.4,
        // 11.2); 200 rows of 2,048 x 2,048 13.3 (13.5, 14.1).
        const int64_t one = tiles(a.rows, p.tile), room = n_cu / one > 1 ? n_cu : 2 * n_cu;
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(room / one, a.inputs / 512));
        p.k_split = (int)ceil_div(ceil_div(a.inputs, p.splits), 64) * 64;
        p.splits = (int)ceil_div(a.inputs, p.k_split);
    } else if (p.tile == k128Wide) {
        // Whole rounds of large tiles; the rows of a last round that would leave most of the device idle go to smaller ones.
        const int64_t wide = ceil_div(a.outputs, kTiles[k128Wide].N), all = tiles(a.rows, k128Wide), whole = all / n_cu * n_cu / wide;
        if (whole && (all - whole * wide) * 2 < n_cu) rows = std::min<int64_t>(rows, whole * kTiles[k128Wide].M);
    }
    size_grid(p, ceil_div(rows, kTiles[p.tile].M), a.outputs, n_cu);
    r.rows = (int)rows;
    if (rows < a.rows) {
        r.rest = p;
        const int64_t left = a.rows - rows;
        r.rest.tile = k64;
        size_grid(r.rest, ceil_div(left, kTiles[r.rest.tile].M), a.outputs, n_cu);
    }
    if (a.adapters) {
        const int64_t of_rows = ceil_div(a.rows, r.joined ? 16 : kTiles[k128].M), of_ranks = ceil_div(a.rank, r.joined ? 32 : kTiles[k128].N);
        // A block takes 1,024 inputs (512, 2,048): one row with rank 16 13.7 (14.1, 14.8), 16 rows of 8 adapters 16.6 (16.3, 19.2), 96 rows of 40
        // with rank 32 into 6,144 33.5 (36.9, 34.1).  In many rows 512 or more (256, 1,024), two row tiles' blocks a CU at most, each with `slots`
        // blocks of its own: 700 rows of 2,048 inputs, ten adapters 40.5 (38.9, 45.6), 12,661 rows 477 (476, 472).
        const int64_t most = std::max<int64_t>(1, r.joined ? a.inputs / 1024 : std::min<int64_t>(a.inputs / 512, 2 * n_cu / (of_rows * of_ranks)));
        r.h_k = (int)ceil_div(ceil_div(a.inputs, most), 64) * 64;
        r.h_splits = (int)ceil_div(a.inputs, r.h_k);
        // 16 blocks share a row tile's adapters (4, 2): 16 rows of 8 adapters 16.6 (19.7, 24.9), 96 of 40 into 6,144 33.5 (39.2, 45.4), but 400 of 64
        // 77 (70, 76).  In many rows 2 (4, 16), made for tiles that hold few requests: 12,661 rows of ten 477 (477, 484), 700 of ten 40.5 (37.4, 38.1).
        // Where each row is a request's, a tile holds many: 512 rows of 64 adapters 188 (144, 115), 96 rows of 40 into 28,672 182 (147, 124).
        r.slots = (int)std::min<int64_t>(a.adapters, r.joined && a.rows <= 512 ? 16 : 2);
        p.shrink = of_rows * of_ranks * r.slots * r.h_splits;
    }
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    r.ws_h2 = a.adapters ? up((int64_t)r.h_splits * a.rows * a.rank * 4) : 0;
    r.ws_unit = r.ws_h2 + (a.adapters && !r.joined ? up((int64_t)a.rows * a.rank * 6) : 0);  // up to three parts
    r.ws_part = r.ws_unit + (a.adapters && !r.joined ? up((int64_t)a.rows * 4) : 0);
    r.ws_bytes = r.ws_part + (r.joined ? (int64_t)p.splits * a.rows * a.outputs * 4 : 0);
    return r;
}

}  // namespace kk
