// Host checks of the products' index arithmetic (kk_product_index.h, the functions that the kernels run).
//   walk: over random launches every tile is taken by exactly one block, and none outside.
//   groups: a group's tiles hold each of its rows once, and the groups' tiles are at most what the launch is sized by.
//   plan: over the range of sizes, accepted launches hold below 2^32 threads, parts cover the inputs, the rows of the two launches
//         are all rows, and the workspace's pieces do not overlap.
//   key: which arguments change the adapters' workspace.
#include <cstdio>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "kk_product_index.h"

using namespace kk;

static int fail(const char* what) {
    std::printf("failed: %s\n", what);
    return 1;
}

static int walk() {
    std::mt19937 g(1);
    for (int n = 0; n < 3000; n++) {
        const int tall = 1 + g() % (n % 3 ? 40 : 700), wide = 1 + g() % 40, blocks = 8 * (1 + g() % 64), total = tall * wide;
        std::vector<int> seen(total);
        for (int b = 0; b < blocks; b++) {
            const TileWalk w = tile_walk(b, blocks, total);
            for (int t = w.first; t < w.end; t += w.step) {
                const TileAt at = tile_at(t, tall, wide);
                if (at.n < 0 || at.n >= wide || at.row < 0 || at.row >= tall) return fail("a tile outside");
                seen[at.row * wide + at.n]++;
            }
        }
        for (int s : seen)
            if (s != 1) return fail("a tile not taken once");
    }
    const int most = 1 << 27;  // the largest launch that is accepted, in its tallest and widest forms
    for (int wide : {1, 7, 8, 9, 1 << 20}) {
        const int tall = most / wide;
        for (int t : {0, 1, tall * wide / 2, tall * wide - 1}) {
            const TileAt at = tile_at(t, tall, wide);
            if (at.n < 0 || at.n >= wide || at.row < 0 || at.row >= tall) return fail("a tile outside a large launch");
        }
    }
    std::printf("walk ok\n");
    return 0;
}

static int groups() {
    std::mt19937 g(2);
    for (int n = 0; n < 3000; n++) {
        const int count = 1 + g() % 70, M = n % 2 ? 64 : 256;
        int start = g() % 3;
        std::vector<int> s{start};
        for (int i = 0; i < count; i++) s.push_back(start += g() % 4 ? g() % (3 * M) : 0);
        const int entries = start + g() % 5;
        int64_t tiles = 0;
        std::vector<int> rows(entries + 1);
        for (int i = 0; i < count; i++) {
            if (!group_ok(s[i], s[i + 1], entries)) return fail("a good group refused");
            const int own = (s[i + 1] - s[i] + M - 1) / M;
            tiles += own;
            for (int j = 0; j < own; j++) {
                Rows r;
                group_rows(s[i], s[i + 1], i, j, M, r);
                if (r.count < 1 || r.count > M || r.first < s[i] || r.first + r.count > s[i + 1]) return fail("rows outside their group");
                for (int k = 0; k < r.count; k++) rows[r.first + k]++;
            }
        }
        for (int i = s[0]; i < start; i++)
            if (rows[i] != 1) return fail("a row not in one tile");
        if (tiles > row_tiles(entries, count, M)) return fail("more tiles than the launch has");
    }
    if (group_ok(-1, 3, 9) || group_ok(4, 3, 9) || group_ok(4, 10, 9) || group_ok(0, INT32_MAX, 9) || group_ok(INT32_MIN, 3, 9)) return fail("a bad group");
    std::printf("groups ok\n");
    return 0;
}

static kk_adapter_product_args adapter(int rows, int in, int out, int adapters, int rank) {
    kk_adapter_product_args a{};
    a.rows = rows, a.inputs = in, a.outputs = out, a.adapters = adapters, a.rank = rank;
    return a;
}

static int plan() {
    std::mt19937 g(3);
    auto size = [&](double top) { return (int)std::exp(std::uniform_real_distribution<double>(0, std::log(top))(g)); };
    int refused = 0, joined = 0, split = 0;
    for (int n = 0; n < 200000; n++) {
        const int n_cu = n % 5 ? 256 : 1 + g() % 300;
        const kk_adapter_product_args a = adapter(size(1 << 24), 8 * size(1 << 12), size(1 << 20), n % 4 ? size(5000) : 0, 8 * (1 + g() % 32));
        const AdapterPlan r = adapter_plan(a, n_cu);
        if (!product_fits(r.main) || !product_fits(r.rest)) {
            refused++;
            continue;
        }
        joined += r.joined, split += r.rows < a.rows;
        for (const ProductPlan* p : {&r.main, &r.rest}) {
            if (p == &r.rest && r.rows == a.rows) continue;
            const int64_t rows = p == &r.main ? r.rows : a.rows - r.rows;
            if (rows < 1 || (int64_t)p->tiles * kTiles[p->tile].M < rows || (int64_t)p->tiles_n * kTiles[p->tile].N < a.outputs) return fail("tiles do not cover");
            if ((int64_t)(p->splits - 1) * p->k_split >= a.inputs || (int64_t)p->splits * p->k_split < a.inputs) return fail("parts do not cover");
            if (p->splits > 1 && p->k_split % 64) return fail("a part's inputs");
            if (p->blocks < 8 || p->blocks % 8 || (p->blocks + p->shrink) * 512 > kMostThreads) return fail("the grid");
        }
        if (r.joined && r.rows != a.rows) return fail("parts of some rows");
        if (a.adapters && ((int64_t)(r.h_splits - 1) * r.h_k >= a.inputs || (int64_t)r.h_splits * r.h_k < a.inputs || r.h_k % 64 || r.slots < 1))
            return fail("the adapters' parts");
        const int64_t h = a.adapters ? (int64_t)r.h_splits * a.rows * a.rank * 4 : 0, h2 = a.adapters && !r.joined ? (int64_t)a.rows * a.rank * 6 : 0;
        if (h > r.ws_h2 || r.ws_h2 + h2 > r.ws_unit || r.ws_unit + (h2 ? (int64_t)a.rows * 4 : 0) > r.ws_part ||
            r.ws_part + (r.joined ? (int64_t)r.main.splits * a.rows * a.outputs * 4 : 0) > r.ws_bytes || r.ws_h2 % 256 || r.ws_unit % 256 || r.ws_part % 256)
            return fail("the workspace");
        if (r.joined && (int64_t)a.rows * ceil_div(a.outputs, 256) * 256 > kMostThreads) return fail("the joining launch");
        kk_expert_product_args e{};
        e.entries = size(1 << 28), e.groups = 1 + g() % 1024, e.inputs = a.inputs, e.outputs = a.outputs, e.gate = n % 3;
        const ProductPlan p = expert_plan(e, n_cu);
        if (product_fits(p) && (p.blocks % 8 || p.blocks < 8 || p.splits != 1 || p.k_split != e.inputs)) return fail("an expert product's grid");
    }
    std::printf("plan ok: refused %d joined %d split %d\n", refused, joined, split);
    return refused > 100000 || !joined || !split;
}

static int key() {
    // 256 CUs; each field changed by itself
    const kk_adapter_product_args a = adapter(300, 4096, 4096, 4, 32);
    const int64_t base = adapter_plan(a, 256).ws_bytes;
    auto differs = [&](const char* name, kk_adapter_product_args b, int n_cu) {
        if (adapter_plan(b, n_cu).ws_bytes != base) std::printf("%s\n", name);
    };
    differs("rows", adapter(301, 4096, 4096, 4, 32), 256);
    differs("inputs", adapter(300, 512, 4096, 4, 32), 256);
    differs("outputs", adapter(300, 4096, 4100, 4, 32), 256);
    differs("adapters", adapter(300, 4096, 4096, 0, 32), 256);
    differs("rank", adapter(300, 4096, 4096, 4, 40), 256);
    differs("compute units", a, 64);
    kk_adapter_product_args b = a;
    std::memset(&b, 0x11, sizeof b);
    b.rows = a.rows, b.inputs = a.inputs, b.outputs = a.outputs, b.adapters = a.adapters, b.rank = a.rank;
    differs("another field", b, 256);
    return 0;
}

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    return what == "walk" ? walk() : what == "groups" ? groups() : what == "plan" ? plan() : what == "key" ? key() : 2;
}
