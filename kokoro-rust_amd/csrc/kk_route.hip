// kk_route.hip -- which experts each row takes, its choices grouped by expert, and the sum of their results.
//
// Choosing.  A row's logits lie on L lanes, J next to each other on each, as 32-bit keys whose order is that of the numbers (0: never
// chosen).  `top` times: the largest key over the lanes, the first lane that holds it, and there its first place, which is the
// lowest expert among equal ones; that key becomes 0.  16 lanes a row up to 256 experts: four rows share a wave's reductions.
// Grouping.  A stable counting sort by expert.  Within 64 choices a lane's rank among those of its expert comes from one ballot for each
// bit of the expert's number; over a block's waves and over blocks from counts.  Nothing depends on the order of atomics.
//
// Few rows take one launch of one block, which is all latency (a row of 64 experts, top 8: 7-8 us);
// many take one that chooses and counts and one that places: 16,384 rows of 128 experts 7.3-8.8 and 7.8-8.6 us, for 5.8 MB.  Both are chains
// of reductions and barriers, not bytes: eight rounds of a row's largest key, and for each 1,024 choices of a block five barriers.
#include <algorithm>

#include "kk_product.h"

namespace kk {
namespace {

constexpr int kRouteThreads = 1024, kRouteWaves = 16;
constexpr int kMostBlocks = 256;  // whose counts every placing block adds up

struct RouteDev {
    const void* logits;
    int64_t logits_row;
    int32_t *expert, *start, *place, *counts;  // counts: [blocks][experts]
    float* weight;
    int rows, experts, top, score, renorm, vec, rows_block, blocks;
    int bits, width;  // bits of experts + 1 numbers; the power of two that holds the experts
    float scale;
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
// Over 16 or 64 lanes, to all of them.
template <int L, class F>
__device__ __forceinline__ uint32_t all_lanes(uint32_t x, F&& f) {
    x = f(x, dpp<0xb1>(x));   // the lane 1 away
    x = f(x, dpp<0x4e>(x));   // 2 away
    x = f(x, dpp<0x141>(x));  // in the other half of 8
    x = f(x, dpp<0x140>(x));  // of 16
    if constexpr (L == 64) {
        const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = f(a[0], a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = f(b[0], b[1]);
    }
    return x;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    return all_lanes<L>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
    return __uint_as_float(all_lanes<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

__device__ __forceinline__ uint32_t key_of(float x) {
    x = fminf(x, 3.402823466e38f) + 0.0f;  // NaN is taken out below; -0 becomes 0
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// Exclusive prefix sums over the block's threads.
__device__ __forceinline__ int block_prefix(int x, int* wave_sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(sum, d);
        if (lane >= d) sum += y;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < wave; i++) before += wave_sums[i];
    return before + sum - x;
}

// Places the choices [from, from + n) of experts at(i), behind base[e] (and counts base up).  count: [17][experts + 1], for the
// waves and their sum.
template <class F>
__device__ __forceinline__ void place_choices(const RouteDev& a, int from, int n, int* base, uint16_t* count, F&& at) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = a.experts + 1;
    for (int p = 0; p < n; p += kRouteThreads) {
        for (int i = tid; i < kRouteWaves * bins; i += kRouteThreads) count[i] = 0;
        const int i = p + tid;
        const bool live = i < n;
        int e = live ? at(i) : 0;
        if (e < 0) e = a.experts;
        uint64_t same = __ballot(live);
        for (int b = 0; b < a.bits; b++) {
            const uint64_t m = __ballot(e >> b & 1);
            same &= e >> b & 1 ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        __syncthreads();
        if (live && rank == 0) count[wave * bins + e] = (uint16_t)__popcll(same);
        __syncthreads();
        for (int j = tid; j < bins; j += kRouteThreads) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < kRouteWaves; w++) {
                const int c = count[w * bins + j];
                count[w * bins + j] = (uint16_t)sum;
                sum += c;
            }
            count[kRouteWaves * bins + j] = (uint16_t)sum;
        }
        __syncthreads();
        if (live) a.place[base[e] + count[wave * bins + e] + rank] = e < a.experts ? from + i : -1;
        __syncthreads();
        for (int j = tid; j < bins; j += kRouteThreads) base[j] += count[kRouteWaves * bins + j];
        __syncthreads();
    }
}

// A block chooses for rows_block rows, kRouteThreads / L at a time.
template <int T, int L, int J>
__global__ void __launch_bounds__(kRouteThreads) choose_kernel(RouteDev a) {
    typedef typename ElemOf<T>::type E;
    constexpr int kAtOnce = kRouteThreads / L, kPer = (KK_MOST_CHOICES + L - 1) / L;
    extern __shared__ int lds[];  // [experts + 1]: counts, then bases; behind them, where there is one block, place_choices' counts
    __shared__ int chosen[kAtOnce][KK_MOST_CHOICES];
    __shared__ float value[kAtOnce][KK_MOST_CHOICES];
    __shared__ int wave_sums[kRouteWaves];
    const int tid = threadIdx.x, sub = tid & (L - 1), slot = tid / L, lane = tid & 63;
    const bool one = a.blocks == 1;
    int* hist = lds;
    for (int i = tid; i < a.experts; i += kRouteThreads) hist[i] = 0;
    __syncthreads();
    const int row0 = blockIdx.x * a.rows_block, row1 = min(a.rows, row0 + a.rows_block);
    for (int at = row0; at < row1; at += kAtOnce) {
        const int row = at + slot;
        const bool live = row < row1;
        const E* x = (const E*)a.logits + (int64_t)min(row, row1 - 1) * a.logits_row;
        E raw[J];
        constexpr int V = 16 / (int)sizeof(E);
        if (J % V == 0 && a.vec) {
#pragma unroll
            for (int j = 0; j + V <= J; j += V) {
                const uint4 q = *(const uint4*)(x + min(sub * J + j, a.experts - V));
                __builtin_memcpy(raw + j, &q, 16);
            }
        } else {
#pragma unroll
            for (int j = 0; j < J; j++) raw[j] = x[min(sub * J + j, a.experts - 1)];
        }
        uint32_t key[J];
        float f[J];
#pragma unroll
        for (int j = 0; j < J; j++) {
            f[j] = ElemOf<T>::load(raw[j]);
            const bool in = sub * J + j < a.experts && f[j] > -INFINITY;  // false for NaN
            key[j] = in ? key_of(f[j]) : 0;
        }
        float sum = 0.0f, most = 0.0f;
        for (int k = 0; k < a.top; k++) {
            uint32_t own = key[0];
#pragma unroll
            for (int j = 1; j < J; j++) own = max(own, key[j]);
            const uint32_t m = lanes_max<L>(own);
            uint64_t who = __ballot(own == m);
            if constexpr (L == 16) who = who >> (lane & 48) & 0xffff;
            if (k == 0) most = m ? of_key(m) : 0.0f;
            if (k == 0 && a.score == KK_SCORE_SOFTMAX) {
#pragma unroll
                for (int j = 0; j < J; j++) sum += key[j] ? expf(of_key(key[j]) - most) : 0.0f;
                sum = lanes_sum<L>(sum);
            }
            if (sub == __ffsll((unsigned long long)who) - 1) {
                int place = -1;
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const bool hit = place < 0 && key[j] == m;
                    place = hit ? j : place;
                    key[j] = hit ? 0 : key[j];
                }
                chosen[slot][k] = m ? sub * J + place : -1;
                value[slot][k] = m ? of_key(m) : 0.0f;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        // Scores in units of exp(unit).  Sigmoids that are divided by their sum have one too, or a row of logits below -88 would have 0 / 0;
        // it ends at -700, about where 64 bits end: a row masked by a type's lowest value has scores, and weights, of 0.
        const bool soft = a.score == KK_SCORE_SOFTMAX;
        const float unit = soft ? most : a.renorm ? fminf(fmaxf(most, -700.0f), 0.0f) : 0.0f;
        auto score = [&](float v) {
            if (!soft && v >= 0.0f) return 1.0f / (1.0f + expf(-v));
            const float x = expf(v - unit);
            return soft ? x : x / (1.0f + expf(v));
        };
        float w[kPer], total = 0.0f;
        int e[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int k = sub + i * L;
            e[i] = k < a.top ? chosen[slot][k] : -1;
            const float v = e[i] >= 0 ? value[slot][k] : 0.0f;
            w[i] = e[i] < 0 ? 0.0f : score(v);
            total += w[i];
        }
        total = lanes_sum<L>(total);
        const float by = a.renorm ? total : soft ? sum : 1.0f;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int k = sub + i * L;
            if (!live || k >= a.top) continue;
            a.expert[(int64_t)row * a.top + k] = e[i];
            a.weight[(int64_t)row * a.top + k] = by > 0.0f ? w[i] / by * a.scale : 0.0f;
            if (e[i] >= 0) atomicAdd(&hist[e[i]], 1);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    const int count = tid < a.experts ? hist[tid] : 0;
    if (!one) {
        if (tid < a.experts) a.counts[(int64_t)blockIdx.x * a.experts + tid] = count;
        return;
    }
    const int before = block_prefix(count, wave_sums);
    __syncthreads();
    if (tid < a.experts) hist[tid] = before, a.start[tid] = before;
    if (tid == a.experts - 1) hist[tid + 1] = before + count, a.start[tid + 1] = before + count;
    __syncthreads();
    // one block has at most kAtOnce rows, whose choices are all in LDS
    place_choices(a, 0, a.rows * a.top, hist, (uint16_t*)(lds + a.experts + 1), [&](int i) {
        const int r = i / a.top;
        return chosen[r][i - r * a.top];
    });
}

__global__ void __launch_bounds__(kRouteThreads) place_kernel(RouteDev a) {
    extern __shared__ int base[];  // [experts + 1], and place_choices' counts
    __shared__ int wave_sums[kRouteWaves];
    __shared__ int parts[2 * kRouteThreads];  // [2][ways][experts]
    const int tid = threadIdx.x;
    uint16_t* count = (uint16_t*)(base + a.experts + 1);
    // an expert's choices in all blocks, and in those before this one: each of `ways` threads adds up every ways-th block
    const int width = a.width, ways = max(1, min(kRouteWaves, kRouteThreads / width)), e = tid & (width - 1), way = tid / width;
    int all = 0, before = 0;
    if (way < ways && e < a.experts) {
        for (int b0 = way; b0 < a.blocks; b0 += 16 * ways) {
            int c[16];
#pragma unroll
            for (int i = 0; i < 16; i++) c[i] = a.counts[min(b0 + i * ways, a.blocks - 1) * a.experts + e];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int b = b0 + i * ways;
                all += b < a.blocks ? c[i] : 0;
                before += b < (int)blockIdx.x ? c[i] : 0;
            }
        }
        if (ways > 1) parts[way * a.experts + e] = all, parts[(ways + way) * a.experts + e] = before;
    }
    __syncthreads();
    if (ways > 1 && tid < a.experts) {
        all = before = 0;
        for (int i = 0; i < ways; i++) all += parts[i * a.experts + tid], before += parts[(ways + i) * a.experts + tid];
    }
    if (tid >= a.experts) all = before = 0;
    const int prefix = block_prefix(all, wave_sums);
    const int row0 = blockIdx.x * a.rows_block, from = row0 * a.top, n = (min(a.rows, row0 + a.rows_block) - row0) * a.top;
    __syncthreads();
    if (tid < a.experts) base[tid] = prefix + before;
    if (tid == a.experts - 1) wave_sums[0] = prefix + all;
    if (blockIdx.x == 0) {
        if (tid < a.experts) a.start[tid] = prefix;
        if (tid == a.experts - 1) a.start[tid + 1] = prefix + all;
    }
    // choices without an expert: all of the blocks before less those that have one
    int own_before = before;
#pragma unroll
    for (int d = 32; d; d >>= 1) own_before += __shfl_xor(own_before, d);
    __syncthreads();
    const int total = wave_sums[0];
    __syncthreads();
    if ((tid & 63) == 0) wave_sums[tid >> 6] = own_before;
    __syncthreads();
    if (tid == 0) {
        int with = 0;
        for (int i = 0; i < kRouteWaves; i++) with += wave_sums[i];
        base[a.experts] = total + from - with;
    }
    __syncthreads();
    place_choices(a, from, n, base, count, [&](int i) { return a.expert[from + i]; });
}

// ------------------------------------------------------------------ the sum of a row's results

struct JoinDev {
    const void *y, *base;
    void* out;
    int64_t y_row, base_row, out_row;
    const int32_t* expert;
    const float* weight;
    int waves, top, values, per_row;  // waves of 64 V values a row
};

// A wave takes 64 V values of a row (V: 16 bytes, or one), so its row, experts and weights are scalars.  Bound by memory: every result is
// read once, kAhead of them in flight a lane: 8,192 rows of 2,048 values, top 8 (327 MB) 54-57 us, 5.7-6.1 TB/s; 64 rows 4.2 us.
template <int T, int V>
__global__ void __launch_bounds__(256) join_kernel(JoinDev a) {
    typedef typename ElemOf<T>::type E;
    constexpr int kAhead = 8;
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (wave >= a.waves) return;
    const int row = wave / a.per_row, at = (wave - row * a.per_row) * (64 * V) + (threadIdx.x & 63) * V;
    const bool in = at < a.values;
    struct Piece {
        E e[V];
    };
    auto load = [&](const void* p, int64_t from) {
        Piece x;
        const E* q = (const E*)p + from + (in ? at : 0);
        if constexpr (V > 1) {
            const uint4 w = stream_load((const uint4*)q);
            __builtin_memcpy(x.e, &w, 16);
        } else {
            x.e[0] = *q;
        }
        return x;
    };
    const int32_t* expert = a.expert + (int64_t)row * a.top;
    const float* weight = a.weight + (int64_t)row * a.top;
    float sum[V] = {};
    Piece base;
    if (a.base) base = load(a.base, row * a.base_row);
    for (int j0 = 0; j0 < a.top; j0 += kAhead) {
        Piece x[kAhead];
        float w[kAhead];
        bool on[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int k = min(j0 + j, a.top - 1);
            on[j] = j0 + j < a.top && expert[k] >= 0;
            w[j] = weight[k];
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (on[j]) x[j] = load(a.y, ((int64_t)row * a.top + j0 + j) * a.y_row);
        if (j0 == 0 && a.base)
#pragma unroll
            for (int k = 0; k < V; k++) sum[k] = ElemOf<T>::load(base.e[k]);
#pragma unroll
        for (int j = 0; j < kAhead; j++)
            if (on[j])
#pragma unroll
                for (int k = 0; k < V; k++) sum[k] = fmaf(w[j], ElemOf<T>::load(x[j].e[k]), sum[k]);
    }
    if (in) store_values<T, V>(a.out, row * a.out_row + at, V > 1, sum);
}

template <int T>
hipError_t run_join(const JoinDev& d, bool vec, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(d.waves, 4)), block(256);
    return vec ? launch(join_kernel<T, T == KK_F32 ? 4 : 8>, grid, block, 0, s, d) : launch(join_kernel<T, 1>, grid, block, 0, s, d);
}

bool join_vec(const kk_expert_join_args& a) {
    const int e = a.type == KK_F32 ? 4 : 2;
    auto whole = [&](const void* p, int64_t row) { return !p || ((uintptr_t)p % 16 == 0 && row * e % 16 == 0); };
    return a.values * (int64_t)e % 16 == 0 && whole(a.y, a.y_row) && whole(a.base, a.base_row) && whole(a.out, a.out_row);
}
int64_t join_per_row(const kk_expert_join_args& a) {
    return ceil_div(a.values, !join_vec(a) ? 64 : a.type == KK_F32 ? 256 : 512);
}

// Rows that a block chooses for, and blocks: few enough that adding up their counts stays short.
void route_blocks(const kk_expert_route_args& a, int& rows_block, int& blocks) {
    const int once = a.experts <= 256 ? kRouteThreads / 16 : kRouteThreads / 64;
    rows_block = (int)ceil_div(ceil_div(std::max(a.rows, 1), kMostBlocks), once) * once;
    blocks = (int)ceil_div(std::max(a.rows, 1), rows_block);
}

template <int T>
hipError_t run_choose(const RouteDev& d, size_t lds, hipStream_t s) {
    const dim3 grid(d.blocks), block(kRouteThreads);
    if (d.experts <= 16) return launch(choose_kernel<T, 16, 1>, grid, block, lds, s, d);
    if (d.experts <= 64) return launch(choose_kernel<T, 16, 4>, grid, block, lds, s, d);
    if (d.experts <= 128) return launch(choose_kernel<T, 16, 8>, grid, block, lds, s, d);
    if (d.experts <= 256) return launch(choose_kernel<T, 16, 16>, grid, block, lds, s, d);
    if (d.experts <= 512) return launch(choose_kernel<T, 64, 8>, grid, block, lds, s, d);
    return launch(choose_kernel<T, 64, 16>, grid, block, lds, s, d);
}

}  // namespace

int64_t route_workspace(const kk_expert_route_args& a) {
    int rows_block, blocks;
    route_blocks(a, rows_block, blocks);
    return blocks == 1 ? 0 : (int64_t)blocks * a.experts * 4;
}

hipError_t launch_route(const kk_expert_route_args& a, hipStream_t s) {
    RouteDev d{};
    d.logits = a.logits, d.logits_row = a.logits_row, d.expert = a.expert, d.start = a.start, d.place = a.place;
    d.counts = (int32_t*)a.workspace, d.weight = a.weight, d.rows = a.rows, d.experts = a.experts, d.top = a.top;
    d.score = a.score, d.renorm = a.renorm, d.scale = a.scale;
    route_blocks(a, d.rows_block, d.blocks);
    while ((1 << d.bits) <= a.experts) d.bits++;
    for (d.width = 1; d.width < a.experts;) d.width *= 2;
    const int e = a.type == KK_F32 ? 4 : 2;
    d.vec = (uintptr_t)a.logits % 16 == 0 && a.logits_row * e % 16 == 0 && a.experts * e % 16 == 0;
    const size_t bins = (size_t)a.experts + 1, lds = bins * 4 + (kRouteWaves + 1) * bins * 2;
    const size_t first = d.blocks == 1 ? lds : bins * 4;
    const hipError_t rc = a.type == KK_BF16 ? run_choose<KK_BF16>(d, first, s)
                          : a.type == KK_F16 ? run_choose<KK_F16>(d, first, s) : run_choose<KK_F32>(d, first, s);
    if (rc != hipSuccess || d.blocks == 1) return rc;
    return launch(place_kernel, dim3(d.blocks), dim3(kRouteThreads), lds, s, d);
}

int64_t join_waves(const kk_expert_join_args& a) { return a.rows * join_per_row(a); }

hipError_t launch_join(const kk_expert_join_args& a, hipStream_t s) {
    JoinDev d{};
    d.y = a.y, d.base = a.base, d.out = a.out, d.y_row = a.y_row, d.base_row = a.base_row, d.out_row = a.out_row;
    d.expert = a.expert, d.weight = a.weight, d.top = a.top, d.values = a.values;
    d.per_row = (int)join_per_row(a), d.waves = (int)join_waves(a);
    const bool vec = join_vec(a);
    if (a.type == KK_BF16) return run_join<KK_BF16>(d, vec, s);
    if (a.type == KK_F16) return run_join<KK_F16>(d, vec, s);
    return run_join<KK_F32>(d, vec, s);
}

}  // namespace kk
