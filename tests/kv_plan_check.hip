// CPU check of how attention over the 8-bit cache is launched (attention_plan in kokoro-rust_amd/csrc/kk_kv_index.h).
//   key    changes one field of random calls at a time and prints the names of those that ever changed the workspace's size
//   fits   random calls over the whole range of sizes: prints "calls N refused R violations V", a violation being a call that is
//          refused although blocks of its kind, whole and of 128 rows, fit into a launch, or whose launches hold 2^32 threads
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <map>
#include <random>
#include <string>

#include "kk_kv_index.h"

using namespace kk;

namespace {

std::mt19937 rng(11);
int below(int n) { return (int)(rng() % (unsigned)n); }
template <class T, size_t N>
T one_of(const T (&x)[N]) {
    return x[below((int)N)];
}

struct Call {
    kk_kv_cache c{};
    kk_kv_batch b{};
    kk_kv_attention_args a{};
    int n_cu = 256;
    int64_t space() const { return attention_plan(c, b, a, n_cu).ws_bytes; }
};

int dim_of() {
    const int d[] = {64, 96, 128, 192, 256};
    return one_of(d);
}

Call some() {
    Call x;
    const int heads[] = {1, 2, 4, 8}, news[] = {1, 1, 2, 5, 9, 40, 200, 1000, 4000}, lens[] = {100, 1000, 8000, 60000};
    x.c.type = 1 + below(2), x.c.heads = one_of(heads), x.c.dim = dim_of(), x.c.pages = 1000;
    x.a.type = 1 + below(2), x.a.heads = 8 * (1 + below(4)), x.a.scale = 0.1f, x.a.causal = below(3) > 0;
    x.a.window = x.a.causal && below(3) == 0 ? 1 + below(3000) : 0;
    x.b.n = 1 + below(below(2) ? 4 : 100), x.b.max_new = one_of(news);
    x.b.rows = x.b.max_new + below(x.b.max_new * (x.b.n - 1) + 1);
    x.b.max_len = std::max(x.b.max_new, one_of(lens)), x.b.table_width = (x.b.max_len + 63) / 64, x.b.table_stride = x.b.table_width;
    return x;
}

int key() {
    static char memory[4096];
    const std::map<std::string, std::function<void(Call&)>> change = {
        {"n", [](Call& x) { x.b.n += 1 + below(50); }},
        {"rows", [](Call& x) { x.b.rows += 1 + below(500); }},
        {"max_new", [](Call& x) { x.b.max_new = 1 + below(x.b.rows); }},
        {"max_len", [](Call& x) { x.b.max_len = x.b.max_new + below(x.b.table_width * 64 - x.b.max_new + 1); }},
        {"cache heads", [](Call& x) { x.c.heads = x.c.heads == 8 ? 1 : 2 * x.c.heads; }},
        {"query heads", [](Call& x) { x.a.heads = x.a.heads == 8 ? 24 : 8; }},
        {"dim", [](Call& x) { x.c.dim = dim_of(); }},
        {"causal", [](Call& x) { x.a.causal = x.a.window ? 1 : !x.a.causal; }},
        {"window", [](Call& x) { x.a.causal = 1, x.a.window = x.a.window ? 0 : 1 + below(3000); }},
        {"compute units", [](Call& x) { x.n_cu = 20 + below(300); }},
        {"cache type", [](Call& x) { x.c.type = 3 - x.c.type; }},
        {"type", [](Call& x) { x.a.type = 3 - x.a.type; }},
        {"pages", [](Call& x) { x.c.pages = 1 + below(1 << 20); }},
        {"table", [](Call& x) { x.b.table_width += 1 + below(9), x.b.table_stride = below(99), x.b.table = (int32_t*)memory; }},
        {"scale", [](Call& x) { x.a.scale = 0.5f; }},
        {"arrays", [](Call& x) {
             x.c.k = x.c.v = memory, x.c.k_scale = x.c.v_scale = (float*)memory, x.c.fault = (int32_t*)memory;
             x.b.row_start = x.b.len = (int32_t*)memory, x.a.q = memory, x.a.out = memory + 8, x.a.workspace = memory;
             x.a.workspace_bytes = 4096;
         }},
        {"strides", [](Call& x) { x.a.q_row = below(999), x.a.q_head = below(99), x.a.out_row = below(999), x.a.out_head = below(99); }},
    };
    for (const auto& [name, f] : change) {
        bool moved = false;
        for (int i = 0; i < 20000; i++) {
            const Call x = some();
            Call y = x;
            f(y);
            if (name == "window" && !x.a.causal) continue;  // two fields at once
            moved |= x.space() != y.space();
        }
        if (moved) std::printf("%s\n", name.c_str());
    }
    return 0;
}

int fits() {
    auto spread = [](int64_t most) { return (int64_t)std::exp2(std::log2((double)most) * below(1 << 20) / (1 << 20)); };
    const uint64_t limit = (uint64_t)1 << 32;
    long calls = 0, refused = 0, bad = 0;
    auto check = [&](const Call& x) {
        const AttnPlan p = attention_plan(x.c, x.b, x.a, x.n_cu);
        const int64_t group = x.a.heads / x.c.heads, rows_heads = (int64_t)x.b.rows * x.a.heads;
        const bool few = (int64_t)x.b.max_new * group <= 32;
        const uint64_t least = (uint64_t)(few ? x.b.n : x.b.rows * group / 128 + x.b.n) * x.c.heads * 256;
        const uint64_t blocks = (uint64_t)p.tiles * x.c.heads * p.parts;
        const uint64_t block = few ? 64 * p.waves : 2 * p.tile_rows;
        const bool ok = attention_fits(p, x.b, x.a.heads, x.c.heads);
        calls++, refused += !ok;
        bad += ok != (least < limit);
        if (ok) bad += blocks * block >= limit || (p.parts > 1 && (uint64_t)(rows_heads + 3) / 4 * 256 >= limit);
        bad += p.chunk < 1 || p.parts < 1 || (p.parts > 1) != (p.ws_bytes > 0);
        return ok;
    };
    for (int i = 0; i < 300000; i++) {
        Call x;
        x.c.dim = dim_of(), x.c.heads = (int)spread(4096), x.a.heads = x.c.heads * (int)spread(4096 / x.c.heads);
        x.a.causal = below(2), x.a.window = x.a.causal && below(2) ? (int)spread(1 << 30) : 0, x.n_cu = 1 + below(400);
        x.b.n = (int)spread(1 << 20), x.b.rows = (int)spread(1 << 28), x.b.max_new = (int)spread(1 << 28);
        x.b.max_len = (int)spread(1 << 30);
        check(x);
    }
    // 2^23 blocks of 512 threads are 2^32: the finer blocks are taken
    Call x;
    x.c.dim = 128, x.c.heads = x.a.heads = 8, x.a.causal = 1;
    x.b.n = (1 << 20) - 1000, x.b.rows = 256000, x.b.max_new = 200, x.b.max_len = 5000;
    bad += !check(x);
    x.b.n--;
    bad += !check(x) || attention_plan(x.c, x.b, x.a, x.n_cu).tile_rows != 256;
    // as many sequences as a batch may have, at the largest bound
    x.b.n = 1 << 20, x.b.rows = 1 << 20, x.b.max_new = 1, x.b.max_len = 1 << 30, x.a.heads = 32;
    bad += !check(x);
    std::printf("calls %ld refused %ld violations %ld\n", calls, refused, bad);
    return 0;
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && !std::strcmp(argv[1], "key")) return key();
    if (argc > 1 && !std::strcmp(argv[1], "fits")) return fits();
    return 2;
}
