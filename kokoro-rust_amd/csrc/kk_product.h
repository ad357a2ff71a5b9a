// kk_product.h -- products of ragged rows (experts, adapters): what their kernels share, and how the host sizes them.
#pragma once
#include <algorithm>
#include <type_traits>

#include "kk_kv.h"

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

struct ProductDev {
    const uint16_t *x, *w;
    int64_t x_row, w_row, w_group;  // in values
    int64_t x_rows, y_rows, y_row;
    const float* bias;
    void* y;
    const int32_t *start, *x_place, *y_place;  // start NULL: one group of all entries
    int32_t* fault;
    double x_inv;  // 1 / x_div
    int entries, groups, inputs, outputs, gate;
    int y_vec;     // 1: 4 outputs in one store, 2: 8
    int tiles, tiles_n, blocks;
    // adapters
    const uint16_t *a, *b;
    const float* scale;
    const int32_t* adapter;
    int adapters, rank;
    int slots, h_splits, h_k;  // blocks that share a row tile's adapters, and its inputs
    float* h;        // [h_splits][rows][rank], times the adapter's scale
    uint16_t* h2;    // [rows][2 rank]: each 8 values' first 16 bits and then what these leave, in units of h_unit[row]
    float* h_unit;   // [rows]
    float* part;     // [splits][entries][outputs]
    int splits, k_split;
};

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
ProductPlan expert_plan(const kk_expert_product_args& a, int n_cu);
AdapterPlan adapter_plan(const kk_adapter_product_args& a, int n_cu);
inline bool product_fits(const ProductPlan& p) {
    return p.shrink * 512 <= kMostThreads / 2 && (int64_t)p.tiles * p.tiles_n * p.splits <= 1 << 28;
}

hipError_t launch_expert_product(const kk_expert_product_args& a, const ProductPlan& p, hipStream_t s);
hipError_t launch_adapter_product(const kk_adapter_product_args& a, const AdapterPlan& p, hipStream_t s);
int64_t route_workspace(const kk_expert_route_args& a);
hipError_t launch_route(const kk_expert_route_args& a, hipStream_t s);
hipError_t launch_join(const kk_expert_join_args& a, hipStream_t s);

}  // namespace kk
