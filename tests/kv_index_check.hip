// CPU check of the index arithmetic of the cache operators (kokoro-rust_amd/csrc/kk_kv_index.h, the functions that the kernels
// run): for random ragged batches, some with planted nonsense (rows that fall, lengths and rows out of range), walks every
// block of a launch and counts violations of
//   - writing and reading back: every (sequence, page) that the batch's good sequences touch belongs to exactly one block, its
//     slots lie in the page, its rows in [0, rows), its page in the table;
//   - attention: every row of a good sequence belongs to exactly one block of each part, the parts of a block's rows cover every
//     page that any of them sees once, their number is at most the plan's, and the pages lie in the table.
// With --plant, tiles start one row late and the check must report violations.  Prints "batches N violations M".
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "kk_kv_index.h"

using namespace kk;

static bool plant = false;

int main(int argc, char** argv) {
    plant = argc > 1 && !std::strcmp(argv[1], "--plant");
    std::mt19937 rng(7);
    auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
    long bad = 0, batches = 0;
    for (int it = 0; it < 3000; it++, batches++) {
        const int n = 1 + below(it % 3 == 0 ? 40 : 4), most = 1 + below(it % 5 == 0 ? 700 : it % 2 ? 5 : 150);
        std::vector<int32_t> start{below(3)}, len;
        for (int b = 0; b < n; b++) {
            const int m = below(6) == 0 ? 0 : b == 0 ? most : below(most + 1);
            start.push_back(start.back() + m);
            len.push_back(below(8) == 0 ? below(m + 1) : m + below(it % 7 == 0 ? 5000 : 200));
        }
        kk_kv_batch h{};
        h.n = n, h.rows = start.back() + below(5), h.max_new = most + below(2);
        for (int x : len) h.max_len = std::max(h.max_len, x);
        h.table_width = (h.max_len + kPage - 1) / kPage + below(2), h.max_len += below(h.table_width * kPage - h.max_len + 1);
        if (it % 4 == 0) {  // nonsense on the device
            const int v[] = {-1, INT32_MIN, INT32_MAX, h.rows + 1, h.max_len + 1};
            for (int k = 0; k < 3; k++) (below(2) ? start[below(n + 1)] : len[below(n)]) = v[below(5)];
        }
        h.row_start = start.data(), h.len = len.data();
        const KvBatchDev B = kv_dev(h);
        bool sane = true;
        for (int b = 0; b < n; b++) {
            KvSeq s;
            sane = kv_seq(B, b, s) && sane;
        }
        auto find = [&](int64_t tile, int64_t G, int M, int E, KvSeq& s) {
            int got = -1;
            for (int b = 0; b < n; b++) {
                KvSeq t;
                int i;
                if (kv_seq(B, b, t) && kv_tile_in(t, tile + plant, G, M, E, i)) got = i, s = t;
            }
            return got;
        };
        // pages
        const KvTiles kt = kv_tiles(h);
        std::vector<int> rows_seen(h.rows, 0);
        for (int64_t x = 0; x < kt.tiles; x++) {
            KvSeq s;
            int i;
            if (kt.per_seq) {
                if (x / kt.per_seq >= n) {
                    bad++;
                    continue;
                }
                i = (int)(x % kt.per_seq) + (plant ? 1 : 0);
                if (!kv_seq(B, (int)(x / kt.per_seq), s)) continue;
            } else if ((i = find(x, 1, kPage, 2, s)) < 0) {
                continue;
            }
            KvPage p;
            if (!kv_page_rows(s, i, p)) continue;
            if (p.lo < 0 || p.hi > kPage || p.lo >= p.hi || p.at < 0 || p.at >= h.table_width) bad++;
            for (int k = p.lo; k < p.hi; k++) {
                const int64_t r = p.row0 + k - p.lo;
                if (r < 0 || r >= h.rows || r - s.r0 != p.at * kPage + k - (s.len - s.m))
                    bad++;
                else
                    rows_seen[r]++;
            }
        }
        if (sane)
            for (int b = 0; b < n; b++)
                for (int r = start[b]; r < start[b + 1]; r++)
                    if (rows_seen[r] != (start[b + 1] - start[b] <= len[b])) bad++;
        // attention
        for (int k = 0; k < 3; k++) {
            kk_kv_cache c{};
            kk_kv_attention_args a{};
            c.heads = 1 + below(8), c.dim = 64;
            const int group = 1 + below(k ? 9 : 2);
            a.heads = c.heads * group;
            a.causal = below(3) > 0, a.window = a.causal && below(2) ? 1 + below(300) : 0;
            const AttnPlan p = attention_plan(c, h, a, 1 + below(300));
            if (p.chunk < 1 || p.parts < 1 || p.parts > kMostParts) bad++;
            std::vector<int> seen((size_t)h.rows * group, 0);
            for (int64_t x = 0; x < p.tiles; x++) {
                KvSeq s;
                int64_t first = 0, end;
                if (p.few) {
                    if (!kv_seq(B, (int)x, s) || s.m == 0) continue;
                    end = (int64_t)s.m * group;
                    if (end > 16 * p.row_tiles) bad++;
                } else {
                    const int i = find(x, group, p.tile_rows, 1, s);
                    const int64_t all = i < 0 ? 0 : (int64_t)s.m * group, tiles = (all + p.tile_rows - 1) / p.tile_rows;
                    if (i < 0 || i >= tiles) continue;
                    first = (int64_t)(tiles - 1 - i) * p.tile_rows, end = std::min(all, first + p.tile_rows);
                }
                for (int64_t r = first; r < end; r++) seen[(size_t)(s.r0 + r / group) * group + r % group]++;
                const int i0 = (int)(first / group), i1 = (int)std::min<int64_t>(s.m - 1, (end - 1) / group);
                const Span sp = span_of(s, a.causal, a.window, p.chunk, i0, i1);
                if (sp.parts > p.parts || sp.lo < 0 || sp.hi > h.table_width || (int64_t)sp.parts * p.chunk < sp.hi - sp.lo) bad++;
                for (int i = i0; i <= i1; i++) {
                    const int pos = s.len - s.m + i;
                    const int hi = a.causal ? std::max(0, std::min(s.len, pos + 1)) : s.len, lo = a.window ? std::max(0, pos - a.window + 1) : 0;
                    if (lo < hi && (lo < sp.lo * kPage || hi > sp.hi * kPage)) bad++;
                }
            }
            if (sane)
                for (int b = 0; b < n; b++)
                    for (int64_t r = (int64_t)start[b] * group; r < (int64_t)start[b + 1] * group; r++)
                        if (seen[r] != 1) bad++;
        }
    }
    std::printf("batches %ld violations %ld\n", batches, bad);
    return 0;
}
