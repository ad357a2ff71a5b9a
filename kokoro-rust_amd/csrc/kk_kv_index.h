// kk_kv_index.h -- which rows, pages and parts the blocks of the cache operators work on: plain index arithmetic, the
// same functions on the host (tests/kv_index_check.hip walks every block of random batches with them) and in the kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kokoro_hip.h"

namespace kk {

constexpr int kPage = KK_KV_PAGE;
// Rows of a (sequence, cache head) up to which attention reads the cache into registers.  17 to 32 rows there against the kernel of many
// rows, us: five drafts of 64 conversations of 1,000 to 4,000 tokens 81 and 188, behind 60,000 tokens 32 and 46; at 256 values
// a head, where two tiles take all 512 registers and 200 bytes of scratch a lane, 154 and 197, 64 and 61: one sequence alone loses
// a little there, a batch gains.
constexpr int kFewRows = 32;
constexpr int kMostParts = 256;  // of the token axis
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1;  // of a launch: HIP counts them in 32 bits

struct KvBatchDev {
    const int32_t *row_start, *len, *table;
    int64_t stride;
    int n, rows, max_new, max_len;
};
inline KvBatchDev kv_dev(const kk_kv_batch& b) {
    return {b.row_start, b.len, b.table, b.table_stride, b.n, b.rows, b.max_new, b.max_len};
}

struct KvSeq {
    int b, r0, m, len;
};

// Sequence b of the batch; false where its rows or its length leave the bounds the launch was sized by.
__host__ __device__ inline bool kv_seq(const KvBatchDev& B, int b, KvSeq& s) {
    s.b = b;
    s.r0 = B.row_start[b];
    const int64_t m = (int64_t)B.row_start[b + 1] - s.r0;
    s.len = B.len[b];
    s.m = (int)m;
    return (s.r0 >= 0) & (m >= 0) & (m <= B.max_new) & (s.r0 + m <= B.rows) & (s.len >= 0) & (s.len <= B.max_len);
}

// A sequence with m rows has at most m G / M + E tiles of M (E = 1 for tiles of its own rows, 2 for pages, where the first
// and the last may be partial), so the tile numbers from floor(r0 G / M) + E b on are its own, without a sum over the
// sequences before it.
__host__ __device__ inline int64_t kv_tile_base(int64_t row, int b, int64_t G, int M, int E) { return row * G / M + (int64_t)E * b; }
__host__ __device__ inline bool kv_tile_in(const KvSeq& s, int64_t tile, int64_t G, int M, int E, int& i) {
    const int64_t base = kv_tile_base(s.r0, s.b, G, M, E);
    i = (int)(tile - base);
    return tile >= base && tile < kv_tile_base((int64_t)s.r0 + s.m, s.b + 1, G, M, E);
}

// ------------------------------------------------------------------ writing and reading back: pages

// `per_seq` > 0: that many block rows for each sequence; 0: tile numbers as above.
struct KvTiles {
    int per_seq;
    int64_t tiles;
};
inline KvTiles kv_tiles(const kk_kv_batch& b) {
    const int64_t per = b.max_new < 2 ? 1 : (b.max_new - 2) / kPage + 2;  // pages that max_new rows can touch
    const int64_t flat = b.rows / kPage + 2 * (int64_t)b.n;
    // A ragged batch of few long and many short sequences would start mostly empty blocks for the longest one's pages; an even
    // one needs no search.  Measured, writing and reading back, us flat against per sequence: two of 8,000 rows among 512 of one 83
    // and 1,106; 64 of one row 13.9 and 11.8.
    if (per * b.n <= 2 * flat) return {(int)per, per * b.n};
    return {0, flat};
}

// Page i of those that a sequence's rows touch: the sequence's page `at`, whose slots [lo, hi) are rows row0...
struct KvPage {
    int at, lo, hi;
    int64_t row0;
};
__host__ __device__ inline bool kv_page_rows(const KvSeq& s, int i, KvPage& p) {
    if (s.m == 0 || s.m > s.len) return false;
    const int first = s.len - s.m;
    p.at = first / kPage + i;
    if (p.at > (s.len - 1) / kPage) return false;
    p.lo = first > p.at * kPage ? first - p.at * kPage : 0;
    p.hi = s.len - p.at * kPage < kPage ? s.len - p.at * kPage : kPage;
    p.row0 = (int64_t)s.r0 + (p.at * kPage + p.lo - first);
    return true;
}

// ------------------------------------------------------------------ attention: parts of the token axis

// What the rows [first, last] (numbers in their sequence) of a block see: pages [lo, hi), in parts of `chunk` pages.
struct Span {
    int lo, hi, parts;
};
__host__ __device__ inline Span span_of(const KvSeq& s, bool causal, int window, int chunk, int first, int last) {
    const int p0 = s.len - s.m + first, p1 = s.len - s.m + last;
    int t_hi = s.len;
    if (causal && p1 + 1 < t_hi) t_hi = p1 + 1 > 0 ? p1 + 1 : 0;
    const int t_lo = window && p0 - window + 1 > 0 ? p0 - window + 1 : 0;
    Span r;
    r.lo = t_lo / kPage;
    r.hi = (t_hi + kPage - 1) / kPage;
    if (r.hi < r.lo) r.hi = r.lo;
    r.parts = r.hi == r.lo ? 1 : (r.hi - r.lo + chunk - 1) / chunk;
    return r;
}

// How kk_kv_attention is launched.
struct AttnPlan {
    bool few;         // at most kFewRows rows of a (sequence, cache head)
    int row_tiles;    // few: 16-row tiles of a block (1 or 2)
    int waves;        // few: of a block, 8 or 4
    int tile_rows;    // rows of a block: many, 256 where that fills the device, or 128
    int threads;      // of a block, at most
    int64_t tiles;    // blocks along the rows
    int chunk, parts; // pages of a part, parts of the axis
    int64_t ws_bytes; // partial results, 0 for one part
};
inline bool join_fits(int64_t rows_heads) { return (rows_heads + 3) / 4 <= kMostThreads / 256; }
inline bool attention_fits(const AttnPlan& p, const kk_kv_batch& b, int heads, int cache_heads) {
    return p.tiles * cache_heads * p.parts <= kMostThreads / p.threads && (p.parts == 1 || join_fits(b.rows * (int64_t)heads));
}
inline AttnPlan attention_plan(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_attention_args& a, int n_cu) {
    AttnPlan p{};
    const int64_t group = a.heads / c.heads, rows = b.max_new * group;
    p.few = rows <= kFewRows;
    p.row_tiles = rows <= 16 ? 1 : 2;
    // tiles of M rows, about: each sequence's last one is half full
    auto about = [&](int M) {
        return std::max<int64_t>(b.n == 1 ? (b.rows * group + M - 1) / M : b.rows * group / M + b.n / 2, 1);
    };
    // pages that a row sees, about
    auto seen = [&](int64_t pages) { return a.causal && !a.window ? pages - b.max_new / (2 * kPage) : pages; };
    // Many rows: 256 a block cost the matrix cores 5% less than 2 x 128 (four prompts of 512 rows behind 8,000 tokens 275 against 295
    // us, one prompt of 4,096 158 against 169), where they fill the device and see enough pages; else the finer blocks end
    // sooner (a prompt of 2,048 57 against 67, 32 prompts of 512 155 against 178, a prompt of 2,500 72 against 80).
    auto tiles = [&](int M) { return b.rows * group / M + b.n; };
    const bool coarse = c.dim <= 128 && about(256) * c.heads >= n_cu && seen(b.max_len / kPage) >= 24 &&
                        tiles(256) * c.heads <= kMostThreads / 512;
    p.tile_rows = p.few ? 16 * p.row_tiles : coarse ? 256 : 128;
    p.tiles = p.few ? b.n : tiles(p.tile_rows);
    int64_t pages = ((int64_t)b.max_len + kPage - 1) / kPage;
    if (a.window) {  // a block's rows stand at most that many tokens apart, and N tokens touch at most N / 64 + 2 pages
        const int64_t tokens = (int64_t)a.window + (p.few ? b.max_new : p.tile_rows / group + 1);
        pages = std::min(pages, tokens / kPage + 2);
    }
    pages = std::max<int64_t>(pages, 1);
    const int64_t blocks = p.tiles * c.heads;
    int64_t chunk = pages;
    // Few rows: a part for each of two blocks a CU where that leaves at least a page a wave (4), and at most 32 pages (more
    // parts than the device holds at once even out ragged lengths).  Measured at 8 heads of 128, us by the parts' pages 4, 8, 16,
    // 32, 64, 128: one sequence of 8,000 tokens 11.2, 12.5, 15.1, 22.2, 34.9, 57.7; of 131,000: 66, 54, 52, 49, 48, 71; 64 of
    // 200 to 8,191: 123, 104, 97, 99, 107, 119; 64 of 8,191: 250, 210, 189, 177, 173, 164.  Up to 1,000 tokens one block's 8
    // waves, without a second launch, are as fast (11.5 against 11.8).
    // Many rows: as many parts as the device holds blocks of at once (two of 128 rows a CU at up to 128 values a head), of 3 pages
    // or more, where the time of the pages saved (0.0094 us a value of the head: 1.2 us a page of 128) is more than the second
    // kernel's 4 us and what the parts write and read.  Measured at 32 heads of 128 over 8, us whole against split: 16 rows behind
    // 8,000 tokens 159 and 20, behind 64,000 1,210 and 52; 100 behind 8,000 162 and 37; two of 512 behind 8,000 235 and 178;
    // where the rule does not split: 700 rows behind 700 36 and 48, 1,024 alone 30 and 46, 1,500 behind 8,000 270 and 281.
    if (p.few) {
        chunk = pages <= 16 ? pages : std::min<int64_t>(std::max<int64_t>((pages * blocks + 2 * n_cu - 1) / (2 * n_cu), 4), 32);
    } else {
        const int64_t fit = (p.tile_rows == 128 && c.dim <= 128 ? 2 : 1) * n_cu;  // blocks that the device holds at once
        const int64_t full = about(p.tile_rows) * c.heads, parts = std::max<int64_t>((fit + full / 16) / full, 1);
        const int64_t part = std::max<int64_t>((pages + parts - 1) / parts, 3);
        const double saved = 0.0094 * c.dim * (double)(seen(pages) - part);
        const double join = 4.0 + 2e-6 * c.dim * (double)((int64_t)b.rows * a.heads * ((pages + part - 1) / part));
        if (part < pages && saved > join) chunk = part;
    }
    // Both launches must hold their blocks (the join's are four (row, head) each): sequences by the hundred thousand get fewer parts.
    int64_t most = std::min<int64_t>(kMostParts, std::max<int64_t>(kMostThreads / (p.few ? 256 : 2 * p.tile_rows) / blocks, 1));
    if (!join_fits(b.rows * (int64_t)a.heads)) most = 1;
    chunk = std::max(chunk, (pages + most - 1) / most);
    p.parts = (int)((pages + chunk - 1) / chunk);
    p.chunk = (int)((pages + p.parts - 1) / p.parts);
    p.parts = (int)((pages + p.chunk - 1) / p.chunk);
    // 8 waves where the blocks leave CUs idle and have the pages: 1,000 tokens of one sequence 10.5 us against 11.9 with 4, of 16
    // 12.1 against 14.6; 4 where blocks share CUs (64 of 1,000: 24.8 against 27.3 with 8).
    p.waves = blocks * p.parts <= n_cu && p.chunk > 4 ? 8 : 4;
    p.threads = p.few ? 64 * p.waves : 2 * p.tile_rows;
    if (p.parts > 1) p.ws_bytes = (int64_t)b.rows * a.heads * p.parts * (c.dim * (int64_t)sizeof(float) + 2 * (int64_t)sizeof(float));
    return p;
}

}  // namespace kk
