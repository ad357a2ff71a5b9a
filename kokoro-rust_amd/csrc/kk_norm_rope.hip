// kk_norm_rope.hip -- RMS norm of each head of q and k and the rotation by position, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w;  pair i of a head turned by pos * f_i
//
// Bound by memory: every value is read and written once (2 x 2 bytes a value in 16 bits).  A head is held by
// L = 2^j lanes; each holds both sides of its pairs (neox: V values at c V and V at rot / 2 + c V), so the rotation
// exchanges nothing between lanes and only the sum of squares is a reduction.  The lanes of a wave hold 64 / L heads
// of one row at once (8 for heads of 128 values in 16 bits) and walk over units (row, 64 / L heads) in order, so a
// row's sines are computed once for its heads.  Angles: pos * f_i / 2 pi in f64, its fraction to f32 and sincospi
// there, which keeps 2^-24 of a turn at any position; a lane's f_i are one f64 exp2 and products, once per wave.
#include <cmath>

#include "kk_kv.h"

namespace kk {
namespace {

struct NormRopeDev {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_row, q_head, k_row, k_head, q_out_row, q_out_head, k_out_row, k_out_head;
    const float *q_weight, *k_weight;
    const int32_t* pos;
    const double* freq;
    double log2_step, step;  // log2(f_1 / f_0) and f_1 / f_0 without a table
    float eps;
    int rows, dim, q_heads, heads, rot, norm;
    int lanes, log2_lanes;   // of a head
    int groups;              // units of a row
    int64_t units, per_wave;
};

// V values a chunk (16 bytes, or 1), K chunk pairs a lane.
template <int T, int V, int K, bool INTER>
__global__ void __launch_bounds__(256) norm_rope_kernel(NormRopeDev a) {
    typedef typename ElemOf<T>::type E;
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t u0 = wave * a.per_wave, u1 = u0 + a.per_wave < a.units ? u0 + a.per_wave : a.units;
    const int sub = lane & (a.lanes - 1), in_wave = lane >> a.log2_lanes, wide = 64 >> a.log2_lanes;
    const int turning = a.rot / (2 * V), pairs = a.dim / (2 * V);  // chunk pairs of a head
    int at[K][2];                                                  // a chunk pair's two places in the head
    double f[K][V];                                                // turns a position of its pairs
#pragma unroll
    for (int j = 0; j < K; j++) {
        const int c = sub + j * a.lanes;
        if (INTER || c >= turning)  // behind `rot` a pair is 2 V values next to each other
            at[j][0] = 2 * V * c, at[j][1] = at[j][0] + V;
        else
            at[j][0] = V * c, at[j][1] = a.rot / 2 + V * c;
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (c >= turning)
                f[j][i] = 0.0;
            else if (a.freq)
                f[j][i] = a.freq[c * V + i] * (0.5 / M_PI);
            else
                f[j][i] = i ? f[j][i - 1] * a.step : exp2(a.log2_step * (double)(c * V)) * (0.5 / M_PI);
        }
    }
    int64_t row_now = -1;
    float cs[K][V], sn[K][V];
    for (int64_t u = u0; u < u1; u++) {
        const int64_t row = u / a.groups;
        const int h = (int)(u - row * a.groups) * wide + in_wave;
        const bool live = h < a.heads, is_q = h < a.q_heads;
        const int hh = is_q ? h : h - a.q_heads;
        const E* x = (const E*)(is_q ? a.q : a.k) + row * (is_q ? a.q_row : a.k_row) + hh * (is_q ? a.q_head : a.k_head);
        float v[K][2 * V];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < K; j++) {
            const bool on = live && sub + j * a.lanes < pairs;
#pragma unroll
            for (int i = 0; i < 2 * V; i++) v[j][i] = 0.0f;
            if (on) {
                load_values<T, V>(x, at[j][0], V > 1, v[j]);
                load_values<T, V>(x, at[j][1], V > 1, v[j] + V);
            }
        }
        if (row != row_now) {
            row_now = row;
            const double pos = (double)a.pos[row];
#pragma unroll
            for (int j = 0; j < K; j++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    double t = pos * f[j][i];
                    t -= rint(t);
                    sincospif(2.0f * (float)t, &sn[j][i], &cs[j][i]);
                }
        }
        if (a.norm) {
#pragma unroll
            for (int j = 0; j < K; j++)
#pragma unroll
                for (int i = 0; i < 2 * V; i++) sum = fmaf(v[j][i], v[j][i], sum);
            for (int m = 1; m < a.lanes; m <<= 1) sum += __shfl_xor(sum, m);
            const float r = 1.0f / sqrtf(sum / (float)a.dim + a.eps);
            const float* w = is_q ? a.q_weight : a.k_weight;
#pragma unroll
            for (int j = 0; j < K; j++) {
                const bool on = w && live && sub + j * a.lanes < pairs;
#pragma unroll
                for (int i = 0; i < 2 * V; i++)
                    v[j][i] *= on ? r * w[at[j][i / V] + i % V] : r;
            }
        }
        E* y = (E*)(is_q ? a.q_out : a.k_out) + row * (is_q ? a.q_out_row : a.k_out_row) +
               hh * (is_q ? a.q_out_head : a.k_out_head);
#pragma unroll
        for (int j = 0; j < K; j++) {
            if (!(live && sub + j * a.lanes < pairs)) continue;
            float o[2 * V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int p = INTER && V > 1 ? 2 * i : i, q = INTER && V > 1 ? 2 * i + 1 : V + i;
                o[p] = v[j][p] * cs[j][i] - v[j][q] * sn[j][i];
                o[q] = v[j][q] * cs[j][i] + v[j][p] * sn[j][i];
            }
            if (sub + j * a.lanes >= turning)  // sine 0 and cosine 1, but for infinities
#pragma unroll
                for (int i = 0; i < 2 * V; i++) o[i] = v[j][i];
            store_values<T, V>(y, at[j][0], V > 1, o);
            store_values<T, V>(y, at[j][1], V > 1, o + V);
        }
    }
}

template <int T>
hipError_t run(NormRopeDev d, bool wide, bool inter, int n_cu, hipStream_t s) {
    constexpr int V = T == KK_F32 ? 4 : 8;
    const int pairs = d.dim / (wide ? 2 * V : 2);
    while (d.lanes < 64 && d.lanes < pairs) d.lanes *= 2, d.log2_lanes++;
    d.groups = (int)ceil_div(d.heads, 64 / d.lanes);
    d.units = (int64_t)d.rows * d.groups;
    // enough waves for every slot (32 a CU), each over several units once there are more
    d.per_wave = ceil_div(d.units, (int64_t)n_cu * 32);
    const dim3 grid((unsigned)ceil_div(ceil_div(d.units, d.per_wave), 4)), block(256);
    // heads have at most 512 values: 64 lanes hold one with 8 or 4 values a chunk, or 4 pairs a lane
    if (wide) return launch(inter ? norm_rope_kernel<T, V, 1, true> : norm_rope_kernel<T, V, 1, false>, grid, block, 0, s, d);
    return launch(inter ? norm_rope_kernel<T, 1, 4, true> : norm_rope_kernel<T, 1, 4, false>, grid, block, 0, s, d);
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
    if (a.rot && !a.freq) {
        d.log2_step = -2.0 / a.rot * std::log2(a.theta);
        d.step = std::exp2(d.log2_step);
    }
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
