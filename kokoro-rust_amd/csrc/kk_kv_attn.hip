// kk_kv_attn.hip -- attention over the 8-bit cache.
//
// Mathematics.  With page scales a (K) and b (V), stored numbers k, v and a row's scale c = scale log2(e):
//   s_t = c a (q . k_t),  out = sum_t 2^{s_t} b v_t / sum_t 2^{s_t}
// in one pass over the pages, keeping per row M, the largest s_t + log2 b seen, and m, the largest s_t (or up to kSlack below them),
//   P_t = 2^{s_t + log2 b - M + kLift},  O = sum P_t v_t = 2^{kLift - M} sum 2^{s_t} b v_t,
//   l = sum_t 2^{s_t - m}: a page's sum of P_t times 2^{M - kLift - log2 b - m},  out = 2^{M - kLift - m} O / l.
// That sum is of P_t in f32, before the rounding to f16 that O's product needs: f16 ends at 2^-24, and a page whose V is small
// beside another's may vanish in O, but its tokens' weights may not in l.
// Folding log2 b into the exponent costs nothing (it goes into the constant of the fused multiply-add) and leaves the
// stored numbers themselves as operands: int8 and e4m3 are exact in f16, so K and V enter the matrix cores without a
// rounding, Q as f16 scaled per row to [2^14, 2^15) (a bf16 value keeps its 8 bits down to 2^-28 of the row's largest), and
// P as f16: 11 bits, and 2^-24 is 2^-35 of the largest P or less (kLift = 11; M lags by kSlack = 4 bits at most, so P <= 2^15).
// f16 rather than bf16 for P because a row that sees one token would otherwise be rounded to 8 bits twice.
// M and m are apart so that scales of V far from 1 stay in range; a page of zeros (b = 0) adds to l alone, its P relative to
// its own largest s.  O and l are rescaled only when M or m move by more than kSlack.
//
// Layout.  Everything is transposed, S^T = K Q^T and O^T = V^T P^T, so that a query row stays on one lane column: its M, m and l are
// one value a lane, a rescale multiplies a lane's own O, and the lanes that compute S hold exactly the P that the second
// product wants, once the 64 tokens of a page are taken in the right order (a sum over tokens may run in any).
#include "kk_kv.h"

namespace kk {
namespace {

constexpr float kSlack = 4.0f, kLift = 11.0f;

struct AttnDev {
    const void* q;
    void* out;
    int64_t q_row, q_head, out_row, out_head;
    float* acc;   // [rows][heads][parts][dim]
    float2* ml;   // [rows][heads][parts]: m and l
    float c;      // scale log2(e)
    int heads, group, type, causal, window, q_vec, out_vec;
    int chunk, parts, tile_rows;
};

__device__ __forceinline__ float other_half(float x, bool maximum) {  // with the lane 32 away
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    return maximum ? fmaxf(a, b) : a + b;
}
__device__ __forceinline__ float other_row(float x, bool maximum) {  // with the lane 16 away
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    return maximum ? fmaxf(a, b) : a + b;
}

// N query values to f16 in units of 2^(e - 14), e the exponent of the row's largest, which `top` holds for the whole row.
__device__ __forceinline__ void q_units(float top, float& down, float& up) {
    int e = (int)(__float_as_uint(top) >> 23) & 255;
    e = min(max(e, 27), 254);
    down = __uint_as_float((uint32_t)(268 - e) << 23);
    up = __uint_as_float((uint32_t)(e - 14) << 23);
}

// P pieces of 8 query values, `step` values apart: all loads before the first is used, and then to f32.
template <int P>
__device__ __forceinline__ void load_query(const AttnDev& a, int64_t at, int step, uint16_t (*e)[8]) {
    const uint16_t* p = (const uint16_t*)a.q + at;
    if (a.q_vec) {
#pragma unroll
        for (int j = 0; j < P; j++) {
            const uint4 w = *(const uint4*)(p + j * step);
            __builtin_memcpy(e[j], &w, 16);
        }
    } else {
#pragma unroll
        for (int j = 0; j < P; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) e[j][k] = p[j * step + k];
    }
}
template <int P>
__device__ __forceinline__ void query_values(const AttnDev& a, const uint16_t (*e)[8], float* x) {
    // a branch, not a choice for each value: code that runs once costs the time to fetch it
    if (a.type == KK_BF16) {
#pragma unroll
        for (int j = 0; j < P; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) x[8 * j + k] = ElemOf<KK_BF16>::load(e[j][k]);
    } else {
#pragma unroll
        for (int j = 0; j < P; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) x[8 * j + k] = ElemOf<KK_F16>::load(e[j][k]);
    }
}

// Four values of a row, next to each other, behind a division by l (or as a part's).
__device__ __forceinline__ void store_out4(const AttnDev& a, int64_t at, const float* x) {
    uint16_t e[4];
    if (a.type == KK_BF16) {
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = ElemOf<KK_BF16>::store(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = ElemOf<KK_F16>::store(x[i]);
    }
    uint16_t* p = (uint16_t*)a.out + at;
    if (a.out_vec) {
        uint2 w;
        __builtin_memcpy(&w, e, 8);
        *(uint2*)p = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = e[i];
    }
}

// A page's number and scales; one that does not exist is page 0 with a NaN scale.
struct PageIn {
    int64_t at;
    float k_scale, v_scale;
    int live;  // slots that hold tokens of the sequence: the bytes of V behind them, which may be the NaN code, are masked
};
__device__ __forceinline__ PageIn page_in(const KvCacheDev& c, const KvSeq& s, int page, int id, int head, bool report) {
    const bool bad = id < 0 || id >= c.pages;
    if (bad) {
        if (report) kv_fault(c, KK_KV_BAD_PAGE);
        id = 0;
    }
    PageIn p;
    p.at = (int64_t)id * c.heads + head;
    p.live = bad ? 0 : s.len - page * kPage;
    p.k_scale = bad ? __uint_as_float(0x7fc00000u) : c.ks[p.at];
    p.v_scale = bad ? 0.0f : c.vs[p.at];  // the scores are NaN: rows that do not see the page stay clean
    return p;
}

// A row's maxima and sum; `page` brings in a page with V's scale b (log_b = log2 b, -inf for a page of zeros), in which the
// row's largest s is `top`.  Returns whether any
// row of the wave moved (then O is to be multiplied by f); P = 2^{s + off}, and the sum of P counts w in l.
struct RowSum {
    float M = -INFINITY, m = -INFINITY, l = 0.0f;
    __device__ __forceinline__ bool page(float log_b, float top, float& f, float& off, float& w) {
        const bool zero = log_b == -INFINITY;
        const float b_log = zero ? 0.0f : log_b;
        const bool up_M = !zero && top + b_log > M + kSlack, up_m = top > m + kSlack;
        const bool moves = __ballot(up_M || up_m) != 0;
        if (moves) {
            const float to_M = up_M ? top + b_log : M, to_m = up_m ? top : m;
            f = up_M ? __builtin_amdgcn_exp2f(M - to_M) : 1.0f;
            if (up_m) l *= __builtin_amdgcn_exp2f(m - to_m);
            M = to_M, m = to_m;
        }
        const float r = zero ? top : M - b_log, ref = r == -INFINITY ? 0.0f : r;
        off = kLift - ref;
        w = __builtin_amdgcn_exp2f(fminf(ref - kLift - (m == -INFINITY ? 0.0f : m), 126.0f));
        return moves;
    }
    // what brings O to units of 2^-m, as l is
    __device__ __forceinline__ float last() const {
        return __builtin_amdgcn_exp2f(M - kLift - (m == -INFINITY ? 0.0f : m));
    }
};

// ------------------------------------------------------------------ few rows: single tokens, drafts

// At most 16 NT rows of a (sequence, cache head).  Bound by reading the cache once.  Each of a block's W waves takes every
// W-th page of the part straight into registers, in 16-byte loads that are the MFMA operands (v_mfma_f32_16x16x32_f16)
// once unpacked; nothing of the cache goes through LDS.  Row i of K's token tile t is token 16 (i / 4) + 4 t + i % 4: then
// lane group g's scores are those of tokens 16 g .. 16 g + 15 in order, the 16 bytes that it loads of each row of V.
// K of the next page is loaded while this one's softmax and second product run, V while its first product runs.  The waves
// leave their O, m and l in LDS, and after one barrier the block's threads join them.
// Measured at 32 heads of 128 over 8: one token each of 64 conversations of 200 to 8,191 tokens (536 MB) 101 us and the join's
// 4.7, 5.1 TB/s over both (a kernel that only reads reaches 6.0, nontemporal, as these loads are, 6.5; with plain ones this
// kernel takes 4% longer, the drafts 8%); five drafts
// behind 131,000 tokens (269 MB) 46 us, 5.9 TB/s, and 4.8; one token behind 500 8 us, a chain of about 15,000 cycles of the
// block's first wave: the sequence 2,100, its loads' addresses 1,300, queries and K 2,000, the one page 3,600, its sums to LDS 700,
// the wait for the wave that ends last 3,500-4,100, and the sums over the waves 1,400.  For 17 to 32 rows each operand of
// the cache feeds two products.
template <int D, int CT, int NT, int W>
__global__ void __launch_bounds__(64 * W, D <= 192 && D * NT <= 256 ? 2 : 1)
attend_few_kernel(KvCacheDev c, KvBatchDev B, AttnDev a) {
    constexpr bool kWide = D % 64 == 0;            // 16 bytes of a K row a lane, else 8
    constexpr int kLoads = kWide ? D / 64 : D / 32;  // of each token tile
    constexpr int kSteps = D / 32, kDim = D / 16;
    constexpr int kLd = D + 4;
    __shared__ float lds_ml[W][NT * 16][2];
    __shared__ __align__(16) float lds_o[W][NT * 16][kLd];
    const int head = blockIdx.x % c.heads, rest = blockIdx.x / c.heads;
    const int part = rest / B.n, b = rest % B.n;  // parts that only long sequences have come last: few blocks end empty meanwhile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    auto number = [&](int page) { return __builtin_amdgcn_readfirstlane(B.table[b * B.stride + page]); };
    // without a window the wave's first page is known before the sequence's length: its number is loaded beside that (the table
    // holds max_len tokens of every sequence; where max_len is 0 there may be none)
    const int guess = part * a.chunk + wave;
    const int early = !a.window && (int64_t)guess * kPage < B.max_len ? B.table[b * B.stride + guess] : 0;
    KvSeq s;
    if (!kv_seq(B, b, s)) {
        if (threadIdx.x == 0 && head == 0 && part == 0) kv_fault(c, KK_KV_BAD_BATCH);
        return;
    }
    if (s.m == 0) return;
    const Span sp = span_of(s, a.causal, a.window, a.chunk, 0, s.m - 1);
    if (part >= sp.parts) return;
    const int page0 = sp.lo + part * a.chunk, page1 = min(page0 + a.chunk, sp.hi);

    // the rows of this lane's columns: their queries are loaded first, so that they are there while K is on its way
    uint16_t raw[NT][D / 32][8] = {};
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = n * 16 + col, i = r / a.group;
        if (i >= s.m) continue;
        const int64_t at = (int64_t)(s.r0 + i) * a.q_row + (head * a.group + r % a.group) * a.q_head;
        if constexpr (kWide) {  // 16 values of each 64 a lane: the two halves of 8 apart
            load_query<D / 64>(a, at + g * 16, 64, raw[n]);
            load_query<D / 64>(a, at + g * 16 + 8, 64, raw[n] + D / 64);
        } else {
            load_query<D / 32>(a, at + g * 8, 32, raw[n]);
        }
    }

    uint4 kr[4][kLoads];
    auto load_k = [&](const PageIn& p) {
        const uint8_t* base = c.k + p.at * (kPage * D);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint8_t* row = base + ((col >> 2) * 16 + t * 4 + (col & 3)) * D;
#pragma unroll
            for (int j = 0; j < kLoads; j++) {
                if constexpr (kWide) {
                    kr[t][j] = stream_load((const uint4*)(row + j * 64 + g * 16));
                } else {
                    const uint2 w = stream_load((const uint2*)(row + j * 32 + g * 8));
                    kr[t][j].x = w.x, kr[t][j].y = w.y;
                }
            }
        }
    };
    const bool report = lane == 0;
    int page = page0 + wave;
    PageIn now;
    if (page < page1) {
        now = page_in(c, s, page, a.window ? number(page) : __builtin_amdgcn_readfirstlane(early), head, report);
        load_k(now);
    }

    f16x8 q[NT][kSteps];
    float qs[NT];
    int lo[NT], hi[NT];  // the tokens that a row sees
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = n * 16 + col, i = r / a.group;
        const bool on = i < s.m;
        float x[D / 4], y[D / 4];
        query_values<D / 32>(a, raw[n], y);
#pragma unroll
        for (int j = 0; j < D / 4; j++) x[j] = kWide ? y[(j / 8 & 1) * (D / 8) + j / 16 * 8 + j % 8] : y[j];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 4; j++) top = fmaxf(top, fabsf(x[j]));
        top = other_half(other_row(top, true), true);
        float down;
        q_units(top, down, qs[n]);
        qs[n] *= a.c;
#pragma unroll
        for (int j = 0; j < kSteps; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) q[n][j][k] = (_Float16)(x[8 * j + k] * down);
        const int pos = s.len - s.m + i;
        hi[n] = on ? (a.causal ? max(0, min(s.len, pos + 1)) : s.len) : 0;
        lo[n] = a.window ? max(0, pos - a.window + 1) : 0;
    }
    // tokens that every row sees
    const int all_lo = a.window ? s.len - a.window : 0, all_hi = a.causal ? s.len - s.m + 1 : s.len;

    f32x4 o[NT][kDim];
    RowSum rs[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int d = 0; d < kDim; d++) o[n][d] = f32x4{0, 0, 0, 0};
    }

    while (page < page1) {
        uint4 vr[kDim];
        {
            const uint8_t* base = c.v + now.at * (kPage * D) + g * 16;
#pragma unroll
            for (int d = 0; d < kDim; d++) vr[d] = stream_load((const uint4*)(base + (d * 16 + col) * kPage));
        }
        f32x4 sc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < 4; t++) sc[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < kLoads; j++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const f16x8 k0 = unpack8<CT>(kr[t][j].x, kr[t][j].y);
                constexpr int kStep = kWide ? 2 : 1;
#pragma unroll
                for (int n = 0; n < NT; n++)
                    sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[n][j * kStep], sc[n][t], 0, 0, 0);
                if constexpr (kWide) {
                    const f16x8 k1 = unpack8<CT>(kr[t][j].z, kr[t][j].w);
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[n][2 * j + 1], sc[n][t], 0, 0, 0);
                }
            }
        const int t0 = page * kPage;
        const PageIn p = now;
        page += W;
        if (page < page1) {
            now = page_in(c, s, page, number(page), head, report);
            load_k(now);
        }
        const bool whole = t0 >= all_lo && t0 + kPage <= all_hi;
        f16x8 pr[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float c1 = qs[n] * p.k_scale;
            if (!whole) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int tok = t0 + g * 16 + t * 4 + r;
                        sc[n][t][r] = tok >= lo[n] && tok < hi[n] ? sc[n][t][r] * c1 : -INFINITY;
                    }
                c1 = 1.0f;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) mx = fmaxf(mx, sc[n][t][r]);
            mx = other_half(other_row(mx, true), true) * c1;
            float f, off, w;
            if (rs[n].page(__builtin_amdgcn_logf(p.v_scale), mx, f, off, w))
#pragma unroll
                for (int d = 0; d < kDim; d++) o[n][d] *= f;
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(sc[n][t][r], c1, off));
                    sum += e;
                    pr[n][t >> 1][(t & 1) * 4 + r] = (_Float16)e;
                }
            rs[n].l = fmaf(sum, w, rs[n].l);
        }
        if (CT == KK_KV_E4M3 && p.live < kPage) {
#pragma unroll
            for (int d = 0; d < kDim; d++) {
                uint32_t* w = (uint32_t*)&vr[d];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int left = p.live - (g * 16 + 4 * i);
                    w[i] = left >= 4 ? w[i] : left <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - 8 * left));
                }
            }
        }
#pragma unroll
        for (int d = 0; d < kDim; d++) {
            const f16x8 v0 = unpack8<CT>(vr[d].x, vr[d].y), v1 = unpack8<CT>(vr[d].z, vr[d].w);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pr[n][0], o[n][d], 0, 0, 0);
                o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pr[n][1], o[n][d], 0, 0, 0);
            }
        }
    }

    const int rows = s.m * a.group;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = n * 16 + col;
        const float l = other_half(other_row(rs[n].l, false), false), f = rs[n].last();
        if (r >= rows) continue;
        if (g == 0) lds_ml[wave][r][0] = rs[n].m, lds_ml[wave][r][1] = l;
#pragma unroll
        for (int d = 0; d < kDim; d++) *(f32x4*)&lds_o[wave][r][d * 16 + g * 4] = o[n][d] * f;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < rows * (D / 4); t += 64 * W) {
        const int r = t / (D / 4), d = t % (D / 4) * 4;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) m = fmaxf(m, lds_ml[w][r][0]);
        const float ref = m == -INFINITY ? 0.0f : m;
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = __builtin_amdgcn_exp2f(lds_ml[w][r][0] - ref);
            l = fmaf(lds_ml[w][r][1], f, l);
            x += *(const f32x4*)&lds_o[w][r][d] * f;
        }
        const int64_t row = s.r0 + r / a.group;
        const int hq = head * a.group + r % a.group;
        if (sp.parts == 1) {
            const float inv = 1.0f / l;
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = l == 0.0f ? 0.0f : x[k] * inv;
            store_out4(a, row * a.out_row + hq * a.out_head + d, y);
        } else {
            const int64_t at = (row * a.heads + hq) * a.parts + part;
            if (d == 0) a.ml[at] = make_float2(m, l);
            *(f32x4*)(a.acc + at * D + d) = x;
        }
    }
}

// ------------------------------------------------------------------ many rows: prompts

// 32 W rows of a (sequence, cache head), 32 a wave (v_mfma_f32_32x32x16_f16).  Bound by the matrix cores and the vector
// instructions beside them (exponentials, unpacking) in about equal parts, so both must run at once.  While a page's scores become
// probabilities, the next page's first product runs, and while its second product runs, the pages after are unpacked, one
// matrix instruction with its share of vector instructions after the other (the order of the source, which sched_barrier
// keeps; left to itself the compiler puts each kind in a row).
// With W = 8 a SIMD's two waves are half a page apart (two barriers a page): one takes its maxima and exponentials while the
// other is in its second product; K and V have three buffers each.  With W = 4, for fewer rows or heads of over 128 values, all waves
// go together, on two buffers.
// A page's bytes are loaded a whole page ahead, unpacked once for all the block's rows and stored to LDS, K by token
// ([token][dim]), V by value ([dim][token]), rows padded by 16 bytes (16-byte reads of 8 lanes then cover all banks).  Within 32
// tokens K's rows are stored so that a lane's 8 scores of one step are 8 tokens in order, as its 16 bytes of V hold them.
// Page numbers and scales are read 64 pages at a time, one a lane.
// Measured: four prompts of 4,096 tokens at 32 heads of 128 over 8 (550 GFLOP) 600-620 us, 887-915 TFLOP/s, 40% of the matrix
// cores' rate at the 2.1 GHz that the device holds meanwhile: in the loop a SIMD takes 1,950 cycles for a wave's page, 1,024 of
// them for its 32 products of 32 cycles; a block's start and end cost another 20,000 (kBufs pages of K
// are unpacked and stored before the first product, which needs one), and half of what the diagonal's pages compute is masked.
// Of 1,000 to 4,096 tokens (278 GFLOP) 327-372 us, 750-850 TFLOP/s.  Four prompts of 2,048 at 16 heads: of 256 values over 4
// 238 us, of 192 over 2 179 us, 576-579 TFLOP/s: 386 to 499 registers leave one wave a SIMD, with nothing to overlap with.  Products and exponentials in turn made 703 TFLOP/s where
// interleaved and half a page apart make 887.  64 rows a wave (half the reads of LDS) were slower, 575 against 740 then: the
// accumulators no longer fit beside the operands and are moved.  l from the unrounded exponentials costs no more than a dot
// instruction over the rounded ones did: 606 us and 606 for the four prompts, e4m3 632 and 654, 430 and 423 at 64 values a head.
template <int D, int CT, int W>
__global__ void __launch_bounds__(64 * W, D <= 128 ? 2 : 1) attend_many_kernel(KvCacheDev c, KvBatchDev B, AttnDev a) {
    constexpr int kRows = 32 * W, kThreads = 64 * W;
    constexpr bool kApart = W == 8;
    constexpr int kBufs = kApart ? 3 : 2;
    constexpr int kK = D + 8, kV = kPage + 8;  // halves of a row in LDS
    constexpr int kKBuf = kPage * kK, kVBuf = D * kV;
    constexpr int kLoads = (4 * D + kThreads - 1) / kThreads;  // 16-byte pieces of K, and of V, a thread (the last one's twice where they do not divide)
    constexpr int kSteps = D / 16, kDim = D / 32;
    constexpr int kFirst = 2 * kSteps, kSecond = 4 * kDim, kAhead = 4;  // products of a page, operands read ahead
    __shared__ __align__(16) _Float16 lds[kBufs * (kKBuf + kVBuf)];
    __shared__ int found[2];
    const int head = blockIdx.x % c.heads, rest = blockIdx.x / c.heads;
    const int part = rest % a.parts;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    KvSeq s;
    int tile = kv_find<kThreads>(c, B, rest / a.parts, a.group, kRows, 1, blockIdx.x == 0, s, found);
    const int64_t all_rows = tile < 0 ? 0 : (int64_t)s.m * a.group;
    const int tiles = (int)((all_rows + kRows - 1) / kRows);
    if (tile < 0 || tile >= tiles) return;
    tile = tiles - 1 - tile;  // the rows that see most first
    const int64_t r_first = (int64_t)tile * kRows;
    const int i_first = (int)(r_first / a.group), over = (int)(r_first % a.group);  // the block's first row: token, head
    const Span sp = span_of(s, a.causal, a.window, a.chunk, i_first, min(s.m - 1, i_first + (over + kRows - 1) / a.group));
    if (part >= sp.parts) return;
    const int page0 = sp.lo + part * a.chunk, page1 = min(page0 + a.chunk, sp.hi);

    // the row of this lane's column, and what the wave's first and last row see; its queries are on their way while the page
    // numbers are read, and the first pages' bytes while the queries are converted
    const int in = over + wave * 32 + col, i = i_first + in / a.group, hq = head * a.group + in % a.group;
    const bool on = i < s.m;
    uint16_t raw[kSteps][8] = {};
    if (on) load_query<kSteps>(a, (int64_t)(s.r0 + i) * a.q_row + hq * a.q_head + h * 8, 16, raw);

    // numbers and scales of the pages from `base` on, one a lane; a page that does not exist is page 0 with a NaN scale of K, and its
    // V is masked: rows that do not see it stay clean
    int base = page0, ids = 0;
    float k_scales = 0.0f, v_logs = 0.0f;
    const int end = page1 - 1;
    auto look = [&](int from) {
        base = from;
        const int id = B.table[s.b * B.stride + min(from + lane, end)];
        const bool bad = id < 0 || id >= c.pages;
        if (bad && wave == 0) kv_fault(c, KK_KV_BAD_PAGE);
        const int64_t at = (int64_t)(bad ? 0 : id) * c.heads + head;
        ids = bad ? -1 : id;
        k_scales = bad ? __uint_as_float(0x7fc00000u) : c.ks[at];
        v_logs = __builtin_amdgcn_logf(bad ? 0.0f : c.vs[at]);
        // waited for here: behind the branch that this is in, the wait would be for every load of the loop
        asm volatile("" ::"v"(ids), "v"(k_scales), "v"(v_logs));
    };
    auto number = [&](int page) { return __builtin_amdgcn_readlane(ids, min(page, end) - base); };
    auto of = [&](float x, int page) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), page - base)); };

    uint4 kr[kLoads], vr[kLoads];
    auto load = [&](uint4* to, const uint8_t* from, int page) {
        const uint8_t* p = from + ((int64_t)max(number(page), 0) * c.heads + head) * (kPage * D);
#pragma unroll
        for (int j = 0; j < kLoads; j++) to[j] = *(const uint4*)(p + (uint32_t)(min(tid + j * kThreads, 4 * D - 1) * 16));
    };
    // half piece n of K (n < 2 kLoads) and then V from their registers to LDS
    auto unpack = [&](int n, _Float16* kb, _Float16* vb) {
        const int j = n / 2 % kLoads, half = n & 1, w = min(tid + j * kThreads, 4 * D - 1);
        if (n < 2 * kLoads) {
            const int tok = w / (D / 16), d = (w % (D / 16)) * 16 + half * 8;
            // token 16 s + 8 h + j of 32 (j = 4 u + k) is the row that lane half h holds as score 8 s + j
            const int row = (tok & 32) | ((tok & 16) | ((tok & 4) << 1) | ((tok & 8) >> 1) | (tok & 3));
            *(f16x8*)(kb + row * kK + d) = half ? unpack8<CT>(kr[j].z, kr[j].w) : unpack8<CT>(kr[j].x, kr[j].y);
        } else {
            *(f16x8*)(vb + w / 4 * kV + w % 4 * 16 + half * 8) = half ? unpack8<CT>(vr[j].z, vr[j].w) : unpack8<CT>(vr[j].x, vr[j].y);
        }
    };
    // slots of V behind the sequence's last token, which may hold the NaN code
    auto mask_v = [&](int page) {
        if constexpr (CT == KK_KV_E4M3) {
            const int live = number(page) < 0 ? 0 : s.len - min(page, end) * kPage;
            if (live >= kPage) return;
#pragma unroll
            for (int j = 0; j < kLoads; j++) {
                const int t = min(tid + j * kThreads, 4 * D - 1) % 4 * 16;
                uint32_t* v = (uint32_t*)&vr[j];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int left = live - (t + 4 * k);
                    v[k] = left >= 4 ? v[k] : left <= 0 ? 0u : v[k] & (0xffffffffu >> (32 - 8 * left));
                }
            }
        }
    };
    _Float16* const k_buf = lds;
    _Float16* const v_buf = lds + kBufs * kKBuf;
    uint4 k_first[kBufs][kLoads], v_first[kBufs][kLoads];
    if (page0 < page1) {
        look(page0);
#pragma unroll
        for (int p = 0; p < kBufs; p++) {
            load(k_first[p], c.k, page0 + p);
            if (p + 1 < kBufs) load(v_first[p], c.v, page0 + p);
        }
    }
    f16x8 q[kSteps];
    float qs;
    {
        float x[D / 2], top = 0.0f;
        query_values<kSteps>(a, raw, x);
#pragma unroll
        for (int j = 0; j < D / 2; j++) top = fmaxf(top, fabsf(x[j]));
        top = other_half(top, true);
        float down;
        q_units(top, down, qs);
        qs *= a.c;
#pragma unroll
        for (int j = 0; j < kSteps; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) q[j][k] = (_Float16)(x[8 * j + k] * down);
    }
    const int off = s.len - s.m;
    const int hi = on ? (a.causal ? max(0, min(s.len, off + i + 1)) : s.len) : 0;
    const int lo = a.window ? max(0, off + i - a.window + 1) : 0;
    const int i0 = i_first + (over + wave * 32) / a.group, i1 = min(s.m - 1, i_first + (over + wave * 32 + 31) / a.group);
    const int all_lo = a.window ? off + i1 - a.window + 1 : 0, all_hi = a.causal ? min(s.len, off + i0 + 1) : s.len;

    f32x16 o[kDim];
#pragma unroll
    for (int d = 0; d < kDim; d++)
#pragma unroll
        for (int k = 0; k < 16; k++) o[d][k] = 0.0f;
    RowSum rs;

    const int k_at = col * kK + h * 8, v_at = col * kV + h * 8;  // of this lane's operands
    // operand n of a page: K's of the first product, then V's of the second
    auto operand = [&](int n, const _Float16* kb, const _Float16* vb) {
        return n < kFirst ? *(const f16x8*)(kb + k_at + (n & 1) * 32 * kK + (n >> 1) * 16)
                          : *(const f16x8*)(vb + v_at + (n - kFirst) % kDim * 32 * kV + (n - kFirst) / kDim * 16);
    };
    int side = 0;  // the page's buffer: page number modulo kBufs, counted from page0
    auto next_side = [](int x) { return x + 1 == kBufs ? 0 : x + 1; };

    // One page: its scores `sc` are there, and the next page's are left in `nx`.  What there is no page for is computed from
    // what the buffers hold and not used.  K of page + kBufs and V of the one before go into the buffers that K of this page
    // and V of the page before were in: all waves have read those (K in the part before, V at least a barrier ago).
    auto one = [&](int page, f32x16* sc, f32x16* nx) {
        const int after = next_side(side);
        const _Float16 *kb = k_buf + after * kKBuf, *vb = v_buf + side * kVBuf;
        if (page + kBufs + 1 - base > 63) look(page);
        if constexpr (kApart) __builtin_amdgcn_s_setprio(1);  // this half takes longer than the other waves' second product
        f16x8 f[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; n++) f[n] = operand(n, kb, vb);
        const int t0 = page * kPage;
        float c1 = qs * of(k_scales, page);
        if (!(t0 >= all_lo && t0 + kPage <= all_hi)) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const int tok = t0 + t * 32 + (k >> 3) * 16 + h * 8 + (k & 7);
                    sc[t][k] = tok >= lo && tok < hi ? sc[t][k] * c1 : -INFINITY;
                }
            c1 = 1.0f;
        }
        float top[4];
#pragma unroll
        for (int k = 0; k < 4; k++) top[k] = fmaxf(sc[k >> 1][8 * (k & 1)], sc[k >> 1][8 * (k & 1) + 1]);
#pragma unroll
        for (int j = 2; j < 8; j += 2)
#pragma unroll
            for (int k = 0; k < 4; k++)
                top[k] = fmaxf(fmaxf(top[k], sc[k >> 1][8 * (k & 1) + j]), sc[k >> 1][8 * (k & 1) + j + 1]);
        const float mx = other_half(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), true) * c1;
        float by, add, w;
        if (rs.page(of(v_logs, page), mx, by, add, w))
#pragma unroll
            for (int d = 0; d < kDim; d++) o[d] *= by;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 16; k++) nx[t][k] = 0.0f;
        f16x8 pr[4];
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < kFirst; n++) {
            nx[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[n % kAhead], q[n >> 1], nx[n & 1], 0, 0, 0);
            f[n % kAhead] = operand(n + kAhead, kb, vb);
#pragma unroll
            for (int k = 16 * n / kFirst; k < 16 * (n + 1) / kFirst; k++) {
                const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[k >> 3][2 * (k & 7)], c1, add));
                const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[k >> 3][2 * (k & 7) + 1], c1, add));
                const f16x2 e = {(_Float16)e0, (_Float16)e1};
                pr[k >> 2][2 * (k & 3)] = e[0], pr[k >> 2][2 * (k & 3) + 1] = e[1];
                sum += e0 + e1;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        rs.l = fmaf(sum, w, rs.l);
        if constexpr (kApart) {
            __builtin_amdgcn_s_setprio(0);
            __syncthreads();
        }
        mask_v(page + kBufs - 1);
        constexpr int kPieces = 4 * kLoads;
        _Float16 *k_to = k_buf + side * kKBuf, *v_to = v_buf + (side == 0 ? kBufs - 1 : side - 1) * kVBuf;
#pragma unroll
        for (int n = 0; n < kSecond; n++) {
            const int d = n % kDim, u = n / kDim;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[(kFirst + n) % kAhead], pr[u], o[d], 0, 0, 0);
            if (n + kAhead < kSecond) f[(kFirst + n) % kAhead] = operand(kFirst + n + kAhead, kb, vb);
#pragma unroll
            for (int k = kPieces * n / kSecond; k < kPieces * (n + 1) / kSecond; k++) unpack(k, k_to, v_to);
            __builtin_amdgcn_sched_barrier(0);
        }
        load(kr, c.k, page + kBufs + 1);
        load(vr, c.v, page + kBufs);
        side = after;
        __syncthreads();
    };

    if (page0 < page1) {
        f32x16 sa[2], sb[2];
#pragma unroll
        for (int p = 0; p < kBufs; p++) {  // K of the first kBufs pages, V of one less
#pragma unroll
            for (int j = 0; j < kLoads; j++) kr[j] = k_first[p][j], vr[j] = v_first[p][j];
            if (p + 1 < kBufs) mask_v(page0 + p);
#pragma unroll
            for (int n = 0; n < (p + 1 < kBufs ? 4 : 2) * kLoads; n++) unpack(n, k_buf + p * kKBuf, v_buf + p * kVBuf);
        }
        load(kr, c.k, page0 + kBufs);
        load(vr, c.v, page0 + kBufs - 1);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 16; k++) sa[t][k] = 0.0f;
#pragma unroll
        for (int n = 0; n < kFirst; n++)
            sa[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(operand(n, k_buf, v_buf), q[n >> 1], sa[n & 1], 0, 0, 0);
        __syncthreads();  // K's first buffer is written again by the first page
        if (kApart && wave >= 4) __syncthreads();
        for (int page = page0;;) {
            one(page, sa, sb);
            if (++page == page1) break;
            one(page, sb, sa);
            if (++page == page1) break;
        }
        if (kApart && wave < 4) __syncthreads();
    }
    const float l = other_half(rs.l, false), last = rs.last();
    if (!on) return;
    const int64_t row = s.r0 + i;
    if (sp.parts == 1) {
        const float inv = l == 0.0f ? 0.0f : last / l;
#pragma unroll
        for (int d = 0; d < kDim; d++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = l == 0.0f ? 0.0f : o[d][u * 4 + k] * inv;
                store_out4(a, row * a.out_row + hq * a.out_head + d * 32 + u * 8 + h * 4, x);
            }
    } else {
        const int64_t at = (row * a.heads + hq) * a.parts + part;
        if (h == 0) a.ml[at] = make_float2(rs.m, l);
#pragma unroll
        for (int d = 0; d < kDim; d++)
#pragma unroll
            for (int u = 0; u < 4; u++)
                *(f32x4*)(a.acc + at * D + d * 32 + u * 8 + h * 4) =
                    f32x4{o[d][u * 4], o[d][u * 4 + 1], o[d][u * 4 + 2], o[d][u * 4 + 3]} * last;
    }
}

// ------------------------------------------------------------------ the parts joined

// out = sum_p 2^{m_p - m} O_p / sum_p 2^{m_p - m} l_p, a wave for each (row, head).  Bound by the latency of three dependent
// loads (the sequence, m, O): 4.7 us for 64 rows of 32 heads in 4 parts as for 5 rows in 64.  Four waves that share the parts were no
// faster: one token behind 1,000,000 tokens, 253 parts, 338 us against 339.
template <int D>
__global__ void __launch_bounds__(256) attend_join_kernel(KvBatchDev B, AttnDev a) {
    constexpr int N = (D + 63) / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = (int64_t)blockIdx.x * 4 + wave;
    const int row = (int)(w / a.heads), hq = (int)(w % a.heads);
    if (row >= B.rows) return;
    KvSeq s;
    bool have = false;
    for (int b0 = 0; b0 < B.n && !have; b0 += 64) {
        KvSeq t{};
        const bool mine = b0 + lane < B.n && kv_seq(B, b0 + lane, t) && row >= t.r0 && row < t.r0 + t.m;
        const uint64_t vote = __ballot(mine);
        if (vote) {
            const int from = __builtin_ctzll(vote);
            have = true;
            s.b = b0 + from, s.r0 = __builtin_amdgcn_readlane(t.r0, from);
            s.m = __builtin_amdgcn_readlane(t.m, from), s.len = __builtin_amdgcn_readlane(t.len, from);
        }
    }
    if (!have) return;
    const int64_t r = (int64_t)(row - s.r0) * a.group + hq % a.group, first = r / a.tile_rows * a.tile_rows;
    const Span sp = span_of(s, a.causal, a.window, a.chunk, (int)(first / a.group),
                            (int)min((int64_t)s.m - 1, (first + a.tile_rows - 1) / a.group));
    if (sp.parts == 1) return;
    const int64_t at = ((int64_t)row * a.heads + hq) * a.parts;
    float m = -INFINITY;
    for (int p = lane; p < sp.parts; p += 64) m = fmaxf(m, a.ml[at + p].x);
    m = other_half(other_row(m, true), true);
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
    const float ref = m == -INFINITY ? 0.0f : m;
    float x[N], l = 0.0f;
#pragma unroll
    for (int k = 0; k < N; k++) x[k] = 0.0f;
    const int dim = min(lane, D - 1 - 64 * (N - 1));  // of the last 64 values
#pragma unroll 8
    for (int p = 0; p < sp.parts; p++) {
        const float2 ml = a.ml[at + p];
        const float f = __builtin_amdgcn_exp2f(ml.x - ref);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int k = 0; k < N; k++) x[k] = fmaf(a.acc[(at + p) * D + (k < N - 1 ? lane : dim) + 64 * k], f, x[k]);
    }
    const float inv = 1.0f / l;
    uint16_t* out = (uint16_t*)a.out + row * a.out_row + hq * a.out_head;
#pragma unroll
    for (int k = 0; k < N; k++)
        if (D % 64 == 0 || lane + 64 * k < D) {
            const float y = l == 0.0f ? 0.0f : x[k] * inv;
            out[lane + 64 * k] = a.type == KK_BF16 ? ElemOf<KK_BF16>::store(y) : ElemOf<KK_F16>::store(y);
        }
}

template <int D, int CT>
hipError_t run(const kk_kv_cache& c, const kk_kv_batch& b, const AttnPlan& p, const AttnDev& a, hipStream_t s) {
    const KvCacheDev cd = kv_dev(c);
    const KvBatchDev bd = kv_dev(b);
    const dim3 grid((unsigned)(p.tiles * c.heads * p.parts));
    hipError_t rc;
    if (!p.few)
        rc = launch(p.tile_rows == 256 ? attend_many_kernel<D, CT, D <= 128 ? 8 : 4> : attend_many_kernel<D, CT, 4>, grid,
                    dim3(2 * p.tile_rows), 0, s, cd, bd, a);
    else if (p.row_tiles == 1 && p.waves == 8)
        rc = launch(attend_few_kernel<D, CT, 1, D <= 192 ? 8 : 4>, grid, dim3(D <= 192 ? 512 : 256), 0, s, cd, bd, a);
    else if (p.row_tiles == 1)
        rc = launch(attend_few_kernel<D, CT, 1, 4>, grid, dim3(256), 0, s, cd, bd, a);
    else
        rc = launch(attend_few_kernel<D, CT, 2, 4>, grid, dim3(256), 0, s, cd, bd, a);
    if (rc != hipSuccess || p.parts == 1) return rc;
    const int64_t sums = (int64_t)b.rows * a.heads;
    return launch(attend_join_kernel<D>, dim3((unsigned)ceil_div(sums, 4)), dim3(256), 0, s, bd, a);
}

}  // namespace

hipError_t launch_kv_attention(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_attention_args& a,
                               const AttnPlan& p, hipStream_t s) {
    AttnDev d{};
    d.q = a.q, d.out = a.out, d.q_row = a.q_row, d.q_head = a.q_head, d.out_row = a.out_row, d.out_head = a.out_head;
    d.acc = (float*)a.workspace;
    if (p.parts > 1) d.ml = (float2*)(d.acc + (int64_t)b.rows * a.heads * p.parts * c.dim);
    d.c = a.scale * 1.44269504f;
    d.heads = a.heads, d.group = a.heads / c.heads, d.type = a.type, d.causal = a.causal, d.window = a.window;
    d.q_vec = (uintptr_t)a.q % 16 == 0 && a.q_row % 8 == 0 && a.q_head % 8 == 0;
    d.out_vec = (uintptr_t)a.out % 8 == 0 && a.out_row % 4 == 0 && a.out_head % 4 == 0;
    d.chunk = p.chunk, d.parts = p.parts, d.tile_rows = p.tile_rows;
#define KK_ATTN_CASE(D) \
    case D: return c.type == KK_KV_INT8 ? run<D, KK_KV_INT8>(c, b, p, d, s) : run<D, KK_KV_E4M3>(c, b, p, d, s);
    switch (c.dim) {
        KK_ATTN_CASE(64)
        KK_ATTN_CASE(96)
        KK_ATTN_CASE(128)
        KK_ATTN_CASE(192)
        KK_ATTN_CASE(256)
    }
#undef KK_ATTN_CASE
    return hipErrorInvalidValue;
}

}  // namespace kk
