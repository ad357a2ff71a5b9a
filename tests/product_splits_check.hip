// Prints how products are launched on 256 CUs (kk_product_index.h): "adapter rows outputs inputs adapters rank" or
// "expert groups entries outputs inputs".
#include <cstdio>
#include <cstdlib>
#include <string>

#include "kk_product_index.h"

using namespace kk;

int main(int argc, char** argv) {
    auto n = [&](int i) { return i < argc ? std::atoi(argv[i]) : 0; };
    if (std::string(argv[1]) == "adapter") {
        kk_adapter_product_args a{};
        a.rows = n(2), a.outputs = n(3), a.inputs = n(4), a.adapters = n(5), a.rank = n(6);
        const AdapterPlan r = adapter_plan(a, 256);
        std::printf("joined %d tile %d rows %d splits %d k_split %d h_splits %d h_k %d fits %d\n", r.joined, r.main.tile, r.rows, r.main.splits,
                    r.main.k_split, r.h_splits, r.h_k, product_fits(r.main) && product_fits(r.rest));
    } else {
        kk_expert_product_args a{};
        a.groups = n(2), a.entries = n(3), a.outputs = n(4), a.inputs = n(5);
        const ProductPlan p = expert_plan(a, 256);
        std::printf("tile %d m %d fits %d\n", p.tile, kTiles[p.tile].M, product_fits(p));
    }
}
