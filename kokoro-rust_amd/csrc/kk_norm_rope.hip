// kk_norm_rope.hip -- RMS norm of each head of q and k and the rotation by position, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w;  pair i of a head turned by pos * f_i
//
// Bound by memory: every value is read and written once (2 x 2 bytes a value in 16 bits).  A head is held by
// L = 2^j lanes; each holds both sides of its pairs (neox: V values at c V and V at rot / 2 + c V), so the rotation
// exchanges nothing between lanes and only the sum of squares is a reduction.  A unit is 64 / L heads of a row (8 heads of
// 128 values in 16 bits); a wave works through a row's units, or some of them where there are few rows, and loads kAhead units
// before it works on the first, which hides the loads' latency without many waves.  The row's angles are computed once: lane i
// takes pair i, pos * f_i / 2 pi in f64, its fraction to f32 and sincospi there (2^-24 of a turn at any position), and
// the wave's lanes read theirs from LDS.
//
// Measured: 16,384 rows of 40 heads of 128 values in 16 bits, 336 MB in 66-71 us, 4.8-5.1 TB/s (a copy of that size moves 5.0-5.3);
// 4,801 rows of 24 heads of 64 in f32, 59 MB in 11.5 us; one row 4.2 us, which is the launch and the latency of its one trip
// to memory.  Before a unit's loads went ahead of the work on the one before (then they waited for each other) the first took 159 us.
// Without 16-byte pieces (an odd address) it takes 245 us: every value is a load of its own.
#include <algorithm>
#include <cmath>

#include "kk_kv.h"

namespace kk {
namespace {

constexpr int kMostPairs = 256;  // of a head: dim <= 512

struct NormRopeDev {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_row, q_head, k_row, k_head, q_out_row, q_out_head, k_out_row, k_out_head;
    const float *q_weight, *k_weight;
    const int32_t* pos;
    const double* freq;
    double log2_step;  // log2(f_1 / f_0) without a table
    float eps;
    int rows, dim, q_heads, heads, rot, norm;
    int lanes, log2_lanes;  // of a head
    int units, split;       // of a row: units, and waves that share them
    int waves;
};

template <int T, int V>
struct Chunk {  // V values next to each other as they lie in memory
    typename ElemOf<T>::type e[V];
    __device__ __forceinline__ void load(const typename ElemOf<T>::type* p) {
        if constexpr (V > 1) {
            const uint4 q = *(const uint4*)p;
            __builtin_memcpy(e, &q, 16);
        } else {
            e[0] = *p;
        }
    }
};

// V values a chunk (16 bytes, or 1), K chunk pairs a lane, kAhead units in flight.
template <int T, int V, int K, int kAhead, bool INTER>
__global__ void __launch_bounds__(256) norm_rope_kernel(NormRopeDev a) {
    typedef typename ElemOf<T>::type E;
    __shared__ __align__(16) float lds[4][2][kMostPairs];
    __shared__ __align__(16) float weight[2][2 * kMostPairs];
    const int lane = threadIdx.x & 63, in_block = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = blockIdx.x * 4 + in_block;
    if (a.norm) {
        for (int i = threadIdx.x; i < a.dim; i += 256) {
            weight[0][i] = a.q_weight ? a.q_weight[i] : 1.0f;
            weight[1][i] = a.k_weight ? a.k_weight[i] : 1.0f;
        }
        __syncthreads();
    }
    if (wave >= a.waves) return;
    float *cos_at = lds[in_block][0], *sin_at = lds[in_block][1];
    const int sub = lane & (a.lanes - 1), slot = lane >> a.log2_lanes, wide = 64 >> a.log2_lanes;
    const int turning = a.rot / (2 * V), pairs = a.dim / (2 * V);  // chunk pairs of a head
    int at[K][2];                                                  // a chunk pair's two places in the head
    bool mine[K];
#pragma unroll
    for (int j = 0; j < K; j++) {
        mine[j] = sub + j * a.lanes < pairs;
        const int c = mine[j] ? sub + j * a.lanes : pairs - 1;  // lanes without one load the last
        if (INTER || c >= turning)                             // behind `rot` a pair is 2 V values next to each other
            at[j][0] = 2 * V * c, at[j][1] = at[j][0] + V;
        else
            at[j][0] = V * c, at[j][1] = a.rot / 2 + V * c;
    }
    const int step = a.waves / a.split, part = wave % a.split;
    const int u0 = a.units * part / a.split, u1 = a.units * (part + 1) / a.split;
    double f[kMostPairs / 64];  // turns a position of the pairs whose angles this lane computes
    bool first = true;
    for (int row = wave / a.split; row < a.rows; row += step) {
        const double pos = (double)a.pos[row];
        float cs[K][V], sn[K][V];
        for (int ub = u0; ub < u1; ub += kAhead) {
            Chunk<T, V> raw[kAhead][K][2];
#pragma unroll
            for (int n = 0; n < kAhead; n++) {
                const int h = min(min(ub + n, u1 - 1) * wide + slot, a.heads - 1);
                const bool is_q = h < a.q_heads;
                const E* x = is_q ? (const E*)a.q + row * a.q_row + h * a.q_head
                                  : (const E*)a.k + row * a.k_row + (h - a.q_heads) * a.k_head;
#pragma unroll
                for (int j = 0; j < K; j++) raw[n][j][0].load(x + at[j][0]), raw[n][j][1].load(x + at[j][1]);
            }
            if (first) {  // behind the first loads
                first = false;
#pragma unroll
                for (int j = 0; j < kMostPairs / 64; j++) {
                    const int i = lane + 64 * j;
                    if (64 * j < a.rot / 2) f[j] = (a.freq ? a.freq[min(i, a.rot / 2 - 1)] : exp2(a.log2_step * (double)i)) * (0.5 / M_PI);
                }
            }
            if (ub == u0) {
#pragma unroll
                for (int j = 0; j < kMostPairs / 64; j++) {
                    if (64 * j >= a.rot / 2) break;
                    double t = pos * f[j];
                    t -= rint(t);
                    float s, c;
                    sincospif(2.0f * (float)t, &s, &c);
                    cos_at[lane + 64 * j] = c, sin_at[lane + 64 * j] = s;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < K; j++) {
                    const int c = min(sub + j * a.lanes, kMostPairs / V - 1);
#pragma unroll
                    for (int i = 0; i < V; i++) cs[j][i] = cos_at[c * V + i], sn[j][i] = sin_at[c * V + i];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int n = 0; n < kAhead; n++) {
                if (ub + n >= u1) break;
                const int h = (ub + n) * wide + slot;
                const bool is_q = h < a.q_heads, live = h < a.heads;
                float v[K][2 * V];
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < K; j++)
#pragma unroll
                    for (int i = 0; i < 2 * V; i++) {
                        v[j][i] = ElemOf<T>::load(raw[n][j][i / V].e[i % V]);
                        const float own = mine[j] ? v[j][i] : 0.0f;  // both factors: an infinity times 0 is NaN
                        sum = fmaf(own, own, sum);
                    }
                if (a.norm) {
                    for (int m = 1; m < a.lanes; m <<= 1) sum += __shfl_xor(sum, m);
                    const float r = 1.0f / sqrtf(sum / (float)a.dim + a.eps);
                    const float* w = weight[is_q ? 0 : 1];
#pragma unroll
                    for (int j = 0; j < K; j++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) v[j][i] *= r * w[at[j][i / V] + i % V];
                }
                E* y = is_q ? (E*)a.q_out + row * a.q_out_row + h * a.q_out_head
                            : (E*)a.k_out + row * a.k_out_row + (h - a.q_heads) * a.k_out_head;
#pragma unroll
                for (int j = 0; j < K; j++) {
                    if (!(live && mine[j])) continue;
                    float* x = v[j];
                    if (sub + j * a.lanes < turning) {
#pragma unroll
                        for (int i = 0; i < V; i++) {
                            const int p = INTER && V > 1 ? 2 * i : i, q = INTER && V > 1 ? 2 * i + 1 : V + i;
                            const float xp = x[p], xq = x[q];
                            x[p] = xp * cs[j][i] - xq * sn[j][i];
                            x[q] = xq * cs[j][i] + xp * sn[j][i];
                        }
                    }
                    store_values<T, V>(y, at[j][0], V > 1, x);
                    store_values<T, V>(y, at[j][1], V > 1, x + V);
                }
            }
        }
    }
}

template <int T>
hipError_t run(NormRopeDev d, bool wide, bool inter, int n_cu, hipStream_t s) {
    constexpr int V = T == KK_F32 ? 4 : 8;
    const int pairs = d.dim / (wide ? 2 * V : 2);
    while (d.lanes < 64 && d.lanes < pairs) d.lanes *= 2, d.log2_lanes++;
    d.units = (int)ceil_div(d.heads, 64 / d.lanes);
    // 16 waves a CU, which with kAhead units each cover the memory's latency; rows that are fewer are shared: one row's five units
    // go to five waves
    const int64_t most = (int64_t)n_cu * 16;
    d.split = (int)std::min<int64_t>(d.units, std::max<int64_t>(1, most / d.rows));
    d.waves = (int)(std::min<int64_t>(d.rows, most / d.split) * d.split);
    const dim3 grid((unsigned)ceil_div(d.waves, 4)), block(256);
    // heads have at most 512 values: 64 lanes hold one with 8 or 4 values a chunk, or with 4 pairs a lane
    if (wide) return launch(inter ? norm_rope_kernel<T, V, 1, 4, true> : norm_rope_kernel<T, V, 1, 4, false>, grid, block, 0, s, d);
    return launch(inter ? norm_rope_kernel<T, 1, 4, 2, true> : norm_rope_kernel<T, 1, 4, 2, false>, grid, block, 0, s, d);
}

}  // namespace

hipError_t launch_norm_rope(const kk_norm_rope& a, int n_cu, hipStream_t s) {
    NormRopeDev d{};
    d.q = a.q, d.k = a.k, d.q_out = a.q_out, d.k_out = a.k_out;
    d.q_row = a.q_row, d.q_head = a.q_head, d.k_row = a.k_row, d.k_head = a.k_head;
    d.q_out_row = a.q_out_row, d.q_out_head = a.q_out_head, d.k_out_row = a.k_out_row, d.k_out_head = a.k_out_head;
    d.q_weight = a.q_weight, d.k_weight = a.k_weight, d.pos = a.pos, d.freq = a.freq;
    d.eps = a.eps, d.rows = a.rows, d.dim = a.dim, d.q_heads = a.q_heads, d.heads = a.q_heads + a.k_heads;
    d.rot = a.rot, d.norm = a.norm, d.lanes = 1, d.log2_lanes = 0;
    if (a.rot && !a.freq) d.log2_step = -2.0 / a.rot * std::log2(a.theta);
    const int e = a.type == KK_F32 ? 4 : 2, V = 16 / e;
    auto whole = [&](int heads, const void* p, int64_t row, int64_t head) {
        return heads == 0 || ((uintptr_t)p % 16 == 0 && row * e % 16 == 0 && head * e % 16 == 0);
    };
    const bool wide = (a.interleaved ? a.rot % (2 * V) == 0 : a.rot / 2 % V == 0) && (a.dim - a.rot) % (2 * V) == 0 &&
                      whole(a.q_heads, a.q, a.q_row, a.q_head) && whole(a.q_heads, a.q_out, a.q_out_row, a.q_out_head) &&
                      whole(a.k_heads, a.k, a.k_row, a.k_head) && whole(a.k_heads, a.k_out, a.k_out_row, a.k_out_head);
    if (a.type == KK_BF16) return run<KK_BF16>(d, wide, a.interleaved, n_cu, s);
    if (a.type == KK_F16) return run<KK_F16>(d, wide, a.interleaved, n_cu, s);
    return run<KK_F32>(d, wide, a.interleaved, n_cu, s);
}

}  // namespace kk
