// kk_product.h -- products of ragged rows (experts, adapters): what their kernels share, and how the host sizes them.
#pragma once
#include <type_traits>

#include "kk_kv.h"
#include "kk_product_index.h"

namespace kk {

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
    int h_rows;      // of the whole call, where a launch takes some
    float* h;        // [h_splits][h_rows][rank], times the adapter's scale
    uint16_t* h2;    // [rows][parts * rank]: each 8 values' first 16 bits, what these leave, and so on, in units of h_unit[row]
    float* h_unit;   // [rows], NaN where h is
    float* part;     // [splits][entries][outputs]
    int splits, k_split;
};

hipError_t launch_expert_product(const kk_expert_product_args& a, const ProductPlan& p, hipStream_t s);
hipError_t launch_adapter_product(const kk_adapter_product_args& a, const AdapterPlan& p, hipStream_t s);
int64_t route_workspace(const kk_expert_route_args& a);
hipError_t launch_route(const kk_expert_route_args& a, hipStream_t s);
int64_t join_waves(const kk_expert_join_args& a);  // of 64 threads
hipError_t launch_join(const kk_expert_join_args& a, hipStream_t s);

}  // namespace kk
