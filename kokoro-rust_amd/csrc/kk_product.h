// kk_product.h -- products of ragged rows (experts, adapters): what their kernels share, and how the host sizes them.
#pragma once
#include "kk_kv.h"

namespace kk {

// Rows `first`..`first + count` (count <= M) of group g.
struct Rows {
    int g, first, count;
};

// Which rows row tile `tile` holds.  A group of m rows has at most m / M + 1 tiles of M, so the numbers from start / M + g on
// are its own, without a sum over the groups before it; some of them stay empty.  Groups that a bad `start` lets overlap may claim one
// tile together: what is left in `i` is then checked against the group as any tile is.
__host__ __device__ inline int64_t row_tiles(int64_t entries, int groups, int M) { return entries / M + groups; }
__host__ __device__ inline bool group_ok(int s0, int s1, int entries) { return s0 >= 0 && s1 >= s0 && s1 <= entries; }
__host__ __device__ inline bool group_has(int s0, int s1, int g, int64_t tile, int M, int& i) {
    const int64_t base = (int64_t)(s0 / M) + g;
    i = (int)(tile - base);
    return tile >= base && tile < (int64_t)(s1 / M) + g + 1;
}
__host__ __device__ inline bool group_rows(int s0, int s1, int g, int i, int M, Rows& r) {
    r.g = g, r.first = s0 + i * M;
    const int left = s1 - r.first;
    r.count = left < M ? left : M;
    return left > 0;
}

struct ProductDev {
    const uint16_t *x, *w;
    int64_t x_row, w_row, w_group;  // in values
    int64_t x_rows, y_rows, y_row;
    const float* bias;
    void* y;
    const int32_t *start, *x_place, *y_place;  // start NULL: one group of all entries
    int32_t* fault;
    int x_div, entries, groups, inputs, outputs, gate;
    int y_vec;     // 8-byte (f32: 16-byte) stores of 4 outputs
    int tiles, tiles_n;
    // adapters
    const uint16_t *a, *b;
    const float* scale;
    const int32_t* adapter;
    int adapters, rank, slots, shrink;
    float* h;           // [rows][rank], times the adapter's scale; or
    uint16_t* h2;       // [rows][2 rank]: each 8 values' first 16 bits and then what these leave, in units of h_unit[row]
    float* h_unit;      // [rows]
    float* part;        // [splits][entries][outputs]
    int splits, k_split;
};

// How a product is launched.
enum { kFew = 0, kTiled = 1 };
struct ProductPlan {
    int kernel;     // kFew: up to 96 rows a block, from memory to registers; kTiled: through LDS
    int M, N, KS;   // rows and outputs of a tile (few rows: of a unit, whose inputs KS waves share)
    int64_t blocks; // of the main kernel
    int splits, k_split;
    bool joined;    // adapters: parts of the main product are summed, and the adapters' share added, by a kernel of their own
    int64_t ws_h, ws_unit, ws_part, ws_bytes;  // workspace
};
ProductPlan expert_plan(const kk_expert_product_args& a, int n_cu);
ProductPlan adapter_plan(const kk_adapter_product_args& a, int n_cu);
inline bool product_fits(const ProductPlan& p) { return p.blocks * 512 <= kMostThreads; }

hipError_t launch_expert_product(const kk_expert_product_args& a, const ProductPlan& p, hipStream_t s);
hipError_t launch_adapter_product(const kk_adapter_product_args& a, const ProductPlan& p, hipStream_t s);
int64_t route_workspace(const kk_expert_route_args& a);
hipError_t launch_route(const kk_expert_route_args& a, hipStream_t s);
hipError_t launch_join(const kk_expert_join_args& a, hipStream_t s);

}  // namespace kk
