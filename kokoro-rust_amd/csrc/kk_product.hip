// kk_product.hip -- products of ragged rows: groups of rows with a matrix each, and a matrix that all rows share beside an
// adapter for each.
//
//   y[i] = act(W_g x[i]),   y[r] = W x[r] + s b (a x[r])
//
// In both kernels the matrix is the MFMA's first operand and the rows are the second, so a lane holds outputs that
// lie next to each other of one row: gathered and scattered rows cost a pointer a lane, and a gate and its partner meet in one lane.
#include "kk_product.h"

namespace kk {
namespace {

template <int T>
struct Mat;
template <>
struct Mat<KK_BF16> {
    static __device__ __forceinline__ f32x16 mul(const uint4& a, const uint4& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mat<KK_F16> {
    static __device__ __forceinline__ f32x16 mul(const uint4& a, const uint4& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, const f32x4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

__device__ __forceinline__ void fault(const ProductDev& p, int bit) {
    if (p.fault) atomicOr(p.fault, bit);
}

// Every thread of a block calls this; false where the tile is empty.
template <int M, int THREADS>
__device__ __forceinline__ bool find_rows(const ProductDev& p, int tile, Rows& r, int* found) {
    if (!p.start) return group_rows(0, p.entries, 0, tile, M, r);
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    for (int g = threadIdx.x; g < p.groups; g += THREADS) {
        const int s0 = p.start[g], s1 = p.start[g + 1];
        int i;
        if (!group_ok(s0, s1, p.entries)) {
            if (blockIdx.x == 0) fault(p, KK_PRODUCT_BAD_START);
        } else if (group_has(s0, s1, g, tile, M, i)) {
            found[0] = g, found[1] = i;
        }
    }
    __syncthreads();
    const int g = __builtin_amdgcn_readfirstlane(found[0]), i = __builtin_amdgcn_readfirstlane(found[1]);
    if (g < 0 || i < 0) return false;
    const int s0 = __builtin_amdgcn_readfirstlane(p.start[g]), s1 = __builtin_amdgcn_readfirstlane(p.start[g + 1]);
    return group_ok(s0, s1, p.entries) && i <= (s1 - s0) / M && group_rows(s0, s1, g, i, M, r);
}

// The row of x of entry e, or -1.
__device__ __forceinline__ int64_t x_of(const ProductDev& p, int e) {
    if (!p.x_place) return e;
    const int place = p.x_place[e];
    if (place < 0 || place / p.x_div >= p.x_rows) {
        fault(p, KK_PRODUCT_BAD_PLACE);
        return -1;
    }
    return place / p.x_div;
}
__device__ __forceinline__ int64_t y_of(const ProductDev& p, int e) {
    if (!p.y_place) return e;
    const int place = p.y_place[e];
    if (place < 0 || place >= p.y_rows) {
        fault(p, KK_PRODUCT_BAD_PLACE);
        return -1;
    }
    return place;
}
__device__ __forceinline__ int adapter_of(const ProductDev& p, int row) {
    const int id = p.adapter[row];
    if (id >= p.adapters) fault(p, KK_PRODUCT_BAD_ADAPTER);
    return id >= p.adapters || id < 0 ? -1 : id;
}

// f(gate) times its partner.  GELU: (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), which loses nothing where tanh nears -1.
__device__ __forceinline__ float gated(int kind, float g, float z) {
    constexpr float kLog2e = 1.44269504089f;
    float u = g;
    if (kind == KK_GATE_GELU) u = 1.5957691216f * fmaf(0.044715f * g * g, g, g);
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * u)) * z;
}

// Up to 4 outputs of a row, next to each other, in the type OUT.
template <int OUT>
__device__ __forceinline__ void store4(void* base, int64_t at, int vec, int left, const float* v) {
    typedef typename ElemOf<OUT>::type E;
    E* p = (E*)base + at;
    E e[4];
#pragma unroll
    for (int i = 0; i < 4; i++) e[i] = ElemOf<OUT>::store(v[i]);
    if (vec && left >= 4) {
        if constexpr (sizeof(E) == 4)
            __builtin_memcpy(__builtin_assume_aligned(p, 16), e, 16);
        else
            __builtin_memcpy(__builtin_assume_aligned(p, 8), e, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) p[i] = e[i];
    }
}

// ------------------------------------------------------------------ few rows

// Up to 16 rows of a group and 16 MT rows of its matrix (8 MT gates and their partners).  Bound by reading the matrix once: each of
// the waves takes every eighth piece of the inputs, in 16-byte loads that are the MFMA operands, and the next piece's loads are under
// way while this one's products run.  The waves leave their sums in LDS, and the block's threads join them.
constexpr int kFewWaves = 8;

template <int T, int MT>
__device__ __forceinline__ void few_sums(const uint16_t* const (&w)[MT], const uint16_t* x, int inputs, int wave, int g, f32x4 (&acc)[MT]) {
    constexpr int J = MT <= 2 ? 4 : MT <= 4 ? 2 : 1, kPiece = 32 * J;  // as many as two sets of registers hold
    uint4 a[2][J][MT], b[2][J];
    auto load = [&](int set, int k0) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int k = k0 + j * 32 + g * 8;
            const bool in = k < inputs;
            b[set][j] = in ? *(const uint4*)(x + k) : uint4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < MT; t++) a[set][j][t] = in ? *(const uint4*)(w[t] + k) : uint4{0, 0, 0, 0};
        }
    };
    auto mul = [&](int set) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = Mat<T>::mul(a[set][j][t], b[set][j], acc[t]);
    };
    constexpr int step = kFewWaves * kPiece;
    int k = wave * kPiece;
    if (k >= inputs) return;
    load(0, k);
    for (; k + step < inputs; k += 2 * step) {
        load(1, k + step);
        mul(0);
        if (k + 2 * step < inputs) load(0, k + 2 * step);
        mul(1);
    }
    if (k < inputs) mul(0);
}

template <int T, int MT, bool GATED, int OUT>
__global__ void __launch_bounds__(64 * kFewWaves) few_kernel(ProductDev p) {
    constexpr int N = 16 * MT, kOut = GATED ? N / 2 : N, kLd = N + 4;
    __shared__ __align__(16) float sums[kFewWaves][16][kLd];
    __shared__ int found[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x / p.tiles_n, n0 = blockIdx.x % p.tiles_n * kOut;
    Rows r;
    if (!find_rows<16, 64 * kFewWaves>(p, tile, r, found)) return;
    const uint16_t* wg = p.w + r.g * p.w_group;
    const uint16_t* w[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const int part = GATED ? t & 1 : 0, o = min(n0 + (GATED ? t >> 1 : t) * 16 + col, p.outputs - 1);
        w[t] = wg + (int64_t)(part * p.outputs + o) * p.w_row;
    }
    const int64_t from = x_of(p, r.first + min(col, r.count - 1));
    f32x4 acc[MT] = {};
    few_sums<T, MT>(w, p.x + max(from, (int64_t)0) * p.x_row, p.inputs, wave, g, acc);
#pragma unroll
    for (int t = 0; t < MT; t++) *(f32x4*)&sums[wave][col][t * 16 + g * 4] = acc[t];
    __syncthreads();
    auto total = [&](int row, int n) {
        f32x4 v = *(const f32x4*)&sums[0][row][n];
#pragma unroll
        for (int i = 1; i < kFewWaves; i++) v += *(const f32x4*)&sums[i][row][n];
        return v;
    };
    const float* bias = p.bias ? p.bias + (int64_t)r.g * p.outputs * (GATED ? 2 : 1) : nullptr;
    for (int t = threadIdx.x; t < r.count * (kOut / 4); t += 64 * kFewWaves) {
        const int row = t / (kOut / 4), o = t % (kOut / 4) * 4, left = p.outputs - (n0 + o);
        if (left <= 0) continue;
        const int e = r.first + row;
        const int64_t to = y_of(p, e);
        if (to < 0 || (p.x_place && x_of(p, e) < 0)) continue;
        f32x4 v = total(row, GATED ? o / 16 * 32 + o % 16 : o);
        if (bias)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] += bias[n0 + o + min(i, left - 1)];
        if constexpr (GATED) {
            f32x4 z = total(row, o / 16 * 32 + 16 + o % 16);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = gated(p.gate, v[i], z[i] + (bias ? bias[p.outputs + n0 + o + min(i, left - 1)] : 0.0f));
        }
        float f[4] = {v[0], v[1], v[2], v[3]};
        store4<OUT>(p.y, to * p.y_row + n0 + o, p.y_vec, left, f);
    }
}

// ------------------------------------------------------------------ many rows

__device__ __forceinline__ void to_lds(const uint16_t* from, uint16_t* to) {  // 16 bytes a lane, in the lanes' order from `to` on
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// BN rows of the matrix and BM rows of x, through LDS in steps of BK inputs, S of them in flight: memory to LDS directly, 16 bytes a
// lane.  A step's row is BK / 8 pieces of 16 bytes, stored in an order that its row number turns (by XOR), so that the 32 rows that an
// operand's lanes read lie on all banks; since the stores go lane after lane, the order is made by what each lane loads.
// WN x WM waves hold BN / WN x BM / WM each in 32 x 32 tiles.  The operands of the next 16 inputs are read while this one's products run.
template <int T, int BN, int BM, int WN, int WM, int BK, int S, int PER_CU, bool GATED, bool EXT, int OUT>
__global__ void __launch_bounds__(64 * WN * WM, PER_CU * WN * WM / 4) tiled_kernel(ProductDev p) {
    constexpr int kWaves = WN * WM, kThreads = 64 * kWaves;
    constexpr int FN = BN / WN / 32, FM = BM / WM / 32, kSub = BK / 16;
    constexpr int kPieces = BK / 8, kRowsIn = 64 / kPieces;  // rows that a wave's load covers
    constexpr int QW = BN / kRowsIn / kWaves, QX = BM / kRowsIn / kWaves, Q = QW + QX;
    static_assert(QW * kRowsIn * kWaves == BN && QX * kRowsIn * kWaves == BM && kSub % 2 == 0, "tile");
    static_assert(!GATED || (FN % 2 == 0 && 32 % kRowsIn == 0), "a gate and its partner in one wave");
    constexpr int kStage = (BN + BM) * BK;
    constexpr int kOutN = GATED ? BN / 2 : BN;
    __shared__ __align__(16) uint16_t lds[S * kStage];
    __shared__ int found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wm = wave / WN;
    // blocks go to the 8 XCDs in turn: an XCD takes tiles that follow each other, which share rows of x and matrices in its L2
    const int per = gridDim.x / 8, t = blockIdx.x % 8 * per + blockIdx.x / 8;
    const int n0 = t % p.tiles_n * kOutN, rest = t / p.tiles_n;
    const int split = rest % p.splits, tile = rest / p.splits;
    Rows r;
    if (tile >= p.tiles || !find_rows<BM, kThreads>(p, tile, r, found)) return;

    const int in_load = lane / kPieces;
    const int piece = (lane % kPieces) ^ (BK == 64 ? in_load & 7 : (in_load >> 1) & 3);  // which one the lane loads
    const uint16_t* wg = p.w + r.g * p.w_group;
    const uint16_t *src[Q];
#pragma unroll
    for (int q = 0; q < QW; q++) {
        const int row = (q * kWaves + wave) * kRowsIn + in_load;
        int64_t o;
        if constexpr (GATED)
            o = min(n0 + row / 64 * 32 + row % 32, p.outputs - 1) + (row & 32 ? p.outputs : 0);
        else
            o = min(n0 + row, p.outputs - 1);
        src[q] = wg + o * p.w_row + piece * 8;
    }
#pragma unroll
    for (int q = 0; q < QX; q++) {
        const int row = (q * kWaves + wave) * kRowsIn + in_load;
        const int64_t from = x_of(p, r.first + min(row, r.count - 1));
        src[QW + q] = p.x + max(from, (int64_t)0) * p.x_row + piece * 8;
    }
    const int k_lo = split * p.k_split, k_hi = min(p.inputs, k_lo + p.k_split);
    const int main_steps = (k_hi - k_lo + BK - 1) / BK;

    // the tile's adapters come first, as more inputs: each one's b beside the rows' h, which is zero in rows of another
    constexpr int kIds = EXT ? (BM + 63) / 64 : 1;
    int ids[kIds], mine[EXT ? QX : 1];  // of the tile's rows, a lane each; and of the rows that this lane loads
    int issue_id = -1, issue_sub = 0, ext_steps = 0;
    const int subs = EXT ? (2 * p.rank + BK - 1) / BK : 0;
    auto next_id = [&](int last) {
        int m = INT32_MAX;
#pragma unroll
        for (int i = 0; i < kIds; i++)
            if (ids[i] > last) m = min(m, ids[i]);
#pragma unroll
        for (int d = 32; d; d >>= 1) m = min(m, __shfl_xor(m, d));
        return __builtin_amdgcn_readfirstlane(m);
    };
    if constexpr (EXT) {
#pragma unroll
        for (int i = 0; i < kIds; i++) ids[i] = i * 64 + lane < r.count ? adapter_of(p, r.first + i * 64 + lane) : -1;
#pragma unroll
        for (int q = 0; q < QX; q++) {
            const int row = (q * kWaves + wave) * kRowsIn + in_load;
            mine[q] = row < r.count ? adapter_of(p, r.first + row) : -1;
        }
        for (int id = next_id(-1); id != INT32_MAX; id = next_id(id)) ext_steps += subs;
        if (ext_steps) issue_id = next_id(-1);
    }
    const int steps = ext_steps + main_steps;

    const uint4 zero = {0, 0, 0, 0};
    auto issue = [&](int step) {
        uint16_t* to = lds + step % S * kStage + wave * (kRowsIn * BK);
        if (EXT && step < ext_steps) {
            const int at = issue_sub * BK + piece * 8;  // of a row of h2, whose b lies at half of it
            const bool in = at < 2 * p.rank;
#pragma unroll
            for (int q = 0; q < QW; q++) {
                const int o = min(n0 + (q * kWaves + wave) * kRowsIn + in_load, p.outputs - 1);
                uint16_t* dst = to + q * kWaves * kRowsIn * BK;
                if (in)
                    to_lds(p.b + ((int64_t)issue_id * p.outputs + o) * p.rank + at / 16 * 8, dst);
                else
                    *(uint4*)(dst + lane * 8) = zero;
            }
#pragma unroll
            for (int q = 0; q < QX; q++) {
                const int row = min((q * kWaves + wave) * kRowsIn + in_load, r.count - 1);
                uint16_t* dst = to + (QW + q) * kWaves * kRowsIn * BK;
                if (in && mine[q] == issue_id)
                    to_lds(p.h2 + (int64_t)(r.first + row) * (2 * p.rank) + at, dst);
                else
                    *(uint4*)(dst + lane * 8) = zero;
            }
            if (++issue_sub == subs) issue_sub = 0, issue_id = next_id(issue_id);
            return;
        }
        const int k0 = k_lo + (step - ext_steps) * BK;
        if (k0 + BK <= k_hi) {
#pragma unroll
            for (int q = 0; q < Q; q++) to_lds(src[q] + k0, to + q * kWaves * kRowsIn * BK);
        } else {
            const bool in = k0 + piece * 8 < k_hi;
#pragma unroll
            for (int q = 0; q < Q; q++) {
                uint16_t* dst = to + q * kWaves * kRowsIn * BK;
                if (in)
                    to_lds(src[q] + k0, dst);
                else
                    *(uint4*)(dst + lane * 8) = zero;
            }
        }
    };
    // All but the last S - 2 steps' loads of this wave, and then of all.  An adapter's step may have fewer loads (a wave whose lanes all
    // store zeros has none), so while one is among those last, all are waited for.
    auto wait = [&](bool all) {
        if (all)
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * Q) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    f32x16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int k = 0; k < 16; k++) acc[i][j][k] = 0.0f;
    uint4 fa[2][FN], fb[2][FM];
    const int col = lane & 31, half = lane >> 5, turn = BK == 64 ? col & 7 : (col >> 1) & 3;
    // operand i of sub-step kk: the matrix's tiles, then the rows'
    auto read = [&](int set, const uint16_t* stage, int kk, int i) {
        const int at = ((kk * 2 + half) ^ turn) * 8;
        if (i < FN)
            fa[set][i] = *(const uint4*)(stage + (wn * (BN / WN) + i * 32 + col) * BK + at);
        else
            fb[set][i - FN] = *(const uint4*)(stage + (BN + wm * (BM / WM) + (i - FN) * 32 + col) * BK + at);
    };

#pragma unroll
    for (int i = 0; i < S - 1; i++)
        if (i < steps) issue(i);
    wait(S - 1 > steps || 1 < ext_steps);
#pragma unroll
    for (int i = 0; i < FN + FM; i++) read(0, lds, 0, i);
    for (int i = 0; i < steps; i++) {
        const uint16_t* stage = lds + i % S * kStage;
        if (EXT && OUT != 0 && T == KK_F16 && i == ext_steps && ext_steps) {
#pragma unroll
            for (int j = 0; j < FM; j++) {
                const int row = r.first + min(wm * (BM / WM) + j * 32 + col, r.count - 1);
                const float unit = adapter_of(p, row) < 0 ? 1.0f : p.h_unit[row];
#pragma unroll
                for (int n = 0; n < FN; n++)
#pragma unroll
                    for (int k = 0; k < 16; k++) acc[n][j][k] *= unit;
            }
        }
        if (i + S - 1 < steps) issue(i + S - 1);
#pragma unroll
        for (int kk = 0; kk < kSub; kk++) {
            const bool last = kk == kSub - 1;
            if (last) {
                if (i + 1 < steps) wait(i + S - 1 >= steps || i + 2 < ext_steps);
                stage = lds + (i + 1) % S * kStage;
            }
            int next = 0;
#pragma unroll
            for (int m = 0; m < FN * FM; m++) {
                acc[m % FN][m / FN] = Mat<T>::mul(fa[kk & 1][m % FN], fb[kk & 1][m / FN], acc[m % FN][m / FN]);
#pragma unroll
                for (; next * (FN * FM) < (m + 1) * (FN + FM); next++) read(~kk & 1, stage, last ? 0 : kk + 1, next);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    const float* bias = p.bias ? p.bias + (int64_t)r.g * p.outputs * (GATED ? 2 : 1) : nullptr;
#pragma unroll
    for (int j = 0; j < FM; j++) {
        const int row = wm * (BM / WM) + j * 32 + col, e = r.first + row;
        if (row >= r.count) continue;
        if constexpr (OUT == 0) {
            float* to = p.part + ((int64_t)split * p.entries + e) * p.outputs;
#pragma unroll
            for (int i = 0; i < FN; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int o = n0 + wn * (BN / WN) + i * 32 + q * 8 + half * 4, left = p.outputs - o;
                    float v[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = acc[i][j][4 * q + k];
                    if (left > 0) store4<KK_F32>(to, o, p.outputs % 4 == 0, left, v);
                }
        } else {
            const int64_t to = y_of(p, e);
            if (to < 0 || (p.x_place && x_of(p, e) < 0)) continue;
#pragma unroll
            for (int i = 0; i < FN; i += GATED ? 2 : 1)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int o = n0 + (wn * (BN / WN) + i * 32) / (GATED ? 2 : 1) + q * 8 + half * 4, left = p.outputs - o;
                    if (left <= 0) continue;
                    float v[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        v[k] = acc[i][j][4 * q + k];
                        if (bias) v[k] += bias[o + min(k, left - 1)];
                        if constexpr (GATED)
                            v[k] = gated(p.gate, v[k], acc[i + 1][j][4 * q + k] + (bias ? bias[p.outputs + o + min(k, left - 1)] : 0.0f));
                    }
                    store4<OUT>(p.y, to * p.y_row + o, p.y_vec, left, v);
                }
        }
    }
}

// ------------------------------------------------------------------ adapters

// h = s a x of 16 rows.  A block takes every slots-th of the adapters that its rows have, its waves pieces of the inputs.
template <int T, int MT>
__global__ void __launch_bounds__(64 * kFewWaves) shrink_kernel(ProductDev p) {
    constexpr int kLd = 16 * MT + 4;
    __shared__ __align__(16) float sums[kFewWaves][16][kLd];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int slot = blockIdx.x % p.slots, first = blockIdx.x / p.slots * 16, count = min(16, p.entries - first);
    const int own = col < count ? adapter_of(p, first + col) : -1;
    const uint16_t* x = p.x + (int64_t)(first + min(col, count - 1)) * p.x_row;
    int id = -1;
    for (int n = 0;; n++) {
        int m = own > id ? own : INT32_MAX;
#pragma unroll
        for (int d = 8; d; d >>= 1) m = min(m, __shfl_xor(m, d));
        id = __builtin_amdgcn_readfirstlane(m);
        if (id == INT32_MAX) return;
        if (n % p.slots != slot) continue;
        const uint16_t* w[MT];
        f32x4 acc[MT] = {};
#pragma unroll
        for (int t = 0; t < MT; t++) w[t] = p.a + ((int64_t)id * p.rank + min(t * 16 + col, p.rank - 1)) * p.inputs;
        few_sums<T, MT>(w, x, p.inputs, wave, g, acc);
        __syncthreads();  // the sums of the adapter before have been read
#pragma unroll
        for (int t = 0; t < MT; t++) *(f32x4*)&sums[wave][col][t * 16 + g * 4] = acc[t];
        __syncthreads();
        // 32 threads a row
        const int row = threadIdx.x >> 5, sub = threadIdx.x & 31;
        const bool on = __shfl(own, row) == id;
        const float s = p.scale[id];
        float v[(MT + 1) / 2], top = 0.0f;
#pragma unroll
        for (int i = 0; i < (MT + 1) / 2; i++) {
            const int k = sub + 32 * i;
            v[i] = 0.0f;
            if (k >= p.rank) continue;
#pragma unroll
            for (int j = 0; j < kFewWaves; j++) v[i] += sums[j][row][k];
            v[i] *= s;
            top = fmaxf(top, fabsf(v[i]));
        }
        if (p.h) {
            if (on)
#pragma unroll
                for (int i = 0; i < (MT + 1) / 2; i++)
                    if (sub + 32 * i < p.rank) p.h[(int64_t)(first + row) * p.rank + sub + 32 * i] = v[i];
            continue;
        }
        float down = 1.0f;
        if constexpr (T == KK_F16) {
            // f16 in units of 2^(e - 14), e the exponent of the row's largest: neither part leaves its range
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
            const int e = min(max((int)(__float_as_uint(top) >> 23) & 255, 27), 254);
            down = __uint_as_float((uint32_t)(268 - e) << 23);
            if (on && sub == 0) p.h_unit[first + row] = __uint_as_float((uint32_t)(e - 14) << 23);
        }
        if (on)
#pragma unroll
            for (int i = 0; i < (MT + 1) / 2; i++) {
                const int k = sub + 32 * i;
                if (k >= p.rank) continue;
                const uint16_t hi = ElemOf<T>::store(v[i] * down);
                uint16_t* to = p.h2 + (int64_t)(first + row) * (2 * p.rank) + k / 8 * 16 + k % 8;
                to[0] = hi;
                to[8] = ElemOf<T>::store(v[i] * down - ElemOf<T>::load(hi));
            }
    }
}

// y = the sum of the parts + bias + b h.  A block takes one row and 1,024 outputs.
template <int T, int OUT>
__global__ void __launch_bounds__(256) expand_kernel(ProductDev p) {
    __shared__ __align__(16) float h[KK_MOST_RANK];
    const int row = blockIdx.x / p.tiles_n, o = blockIdx.x % p.tiles_n * 1024 + threadIdx.x * 4, left = p.outputs - o;
    const int id = p.adapters ? adapter_of(p, row) : -1;
    if (id >= 0)
        for (int i = threadIdx.x; i < p.rank; i += 256) h[i] = p.h[(int64_t)row * p.rank + i];
    __syncthreads();
    if (left <= 0) return;
    float v[4] = {};
    const bool whole = p.outputs % 4 == 0;
    for (int s = 0; s < p.splits; s++) {
        const float* from = p.part + ((int64_t)s * p.entries + row) * p.outputs + o;
        if (whole) {
            const f32x4 q = *(const f32x4*)from;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] += q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] += from[min(i, left - 1)];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (p.bias) v[i] += p.bias[o + min(i, left - 1)];
        if (id < 0) continue;
        const uint16_t* b = p.b + ((int64_t)id * p.outputs + o + min(i, left - 1)) * p.rank;
        for (int k = 0; k < p.rank; k += 8) {
            const uint4 q = *(const uint4*)(b + k);
            uint16_t e[8];
            __builtin_memcpy(e, &q, 16);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i] = fmaf(ElemOf<T>::load(e[j]), h[k + j], v[i]);
        }
    }
    store4<OUT>(p.y, (int64_t)row * p.y_row + o, p.y_vec, left, v);
}

// ------------------------------------------------------------------ launches

template <int T, bool GATED, bool EXT, int OUT>
hipError_t run_tiled(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)((p.blocks + 7) / 8 * 8)), block(256);
    if (p.M == 256) return launch(tiled_kernel<T, 256, 256, 2, 2, 32, 4, 1, GATED, EXT, OUT>, grid, block, 0, s, d);
    if (p.M == 128) return launch(tiled_kernel<T, 128, 128, 2, 2, 32, 4, 2, GATED, EXT, OUT>, grid, block, 0, s, d);
    return launch(tiled_kernel<T, 128, 64, 2, 2, 32, 4, 2, GATED, EXT, OUT>, grid, block, 0, s, d);
}

template <int T, bool GATED, int OUT>
hipError_t run_few(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)p.blocks), block(64 * kFewWaves);
    constexpr int kTwo = GATED ? 2 : 1;
    if (p.N == 16) return launch(few_kernel<T, kTwo, GATED, OUT>, grid, block, 0, s, d);
    return launch(few_kernel<T, 2 * kTwo, GATED, OUT>, grid, block, 0, s, d);
}

template <int T>
hipError_t run_shrink(const ProductDev& d, hipStream_t s) {
    const dim3 grid((unsigned)(ceil_div(d.entries, 16) * d.slots)), block(64 * kFewWaves);
    if (d.rank <= 16) return launch(shrink_kernel<T, 1>, grid, block, 0, s, d);
    if (d.rank <= 32) return launch(shrink_kernel<T, 2>, grid, block, 0, s, d);
    if (d.rank <= 64) return launch(shrink_kernel<T, 4>, grid, block, 0, s, d);
    if (d.rank <= 128) return launch(shrink_kernel<T, 8>, grid, block, 0, s, d);
    return launch(shrink_kernel<T, 16>, grid, block, 0, s, d);
}

}  // namespace

ProductPlan expert_plan(const kk_expert_product_args& a, int n_cu) {
    ProductPlan p{};
    p.splits = 1, p.k_split = a.inputs;
    const int64_t wide = (int64_t)a.outputs * (a.gate != KK_GATE_NONE ? 2 : 1), mean = a.entries / a.groups;
    if (mean <= 16) {
        p.kernel = kFew, p.M = 16, p.N = 32;
        p.blocks = row_tiles(a.entries, a.groups, 16) * ceil_div(a.outputs, p.N);
        return p;
    }
    p.kernel = kTiled;
    p.M = mean >= 512 ? 256 : mean >= 96 ? 128 : 64;
    p.N = p.M == 256 ? 256 : 128;
    p.blocks = row_tiles(a.entries, a.groups, p.M) * ceil_div(wide, p.N);
    return p;
}

ProductPlan adapter_plan(const kk_adapter_product_args& a, int n_cu) {
    ProductPlan p{};
    p.splits = 1, p.k_split = a.inputs;
    p.kernel = kTiled;
    auto tiles = [&](int M, int N) { return ceil_div(a.rows, M) * ceil_div(a.outputs, N); };
    p.M = 64;
    for (int m : {128, 256})
        if (tiles(m, m) >= n_cu) p.M = m;
    p.N = p.M == 256 ? 256 : 128;
    p.blocks = tiles(p.M, p.N);
    if (p.blocks < n_cu) {
        p.joined = true;
        p.splits = (int)std::min<int64_t>(ceil_div(2 * n_cu, p.blocks), std::max<int64_t>(1, a.inputs / 256));
        p.k_split = (int)ceil_div(ceil_div(a.inputs, p.splits), 64) * 64;
        p.splits = (int)ceil_div(a.inputs, p.k_split);
        p.blocks *= p.splits;
    }
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    p.ws_h = 0;
    p.ws_unit = a.adapters ? up((int64_t)a.rows * a.rank * 4) : 0;
    p.ws_part = p.ws_unit + (a.adapters && !p.joined ? up((int64_t)a.rows * 4) : 0);
    p.ws_bytes = p.ws_part + (p.joined ? (int64_t)p.splits * a.rows * a.outputs * 4 : 0);
    return p;
}

template <int T>
static hipError_t expert_run(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    if (p.kernel == kFew) return d.gate ? run_few<T, true, T>(d, p, s) : run_few<T, false, T>(d, p, s);
    return d.gate ? run_tiled<T, true, false, T>(d, p, s) : run_tiled<T, false, false, T>(d, p, s);
}

hipError_t launch_expert_product(const kk_expert_product_args& a, const ProductPlan& p, hipStream_t s) {
    ProductDev d{};
    d.x = (const uint16_t*)a.x, d.w = (const uint16_t*)a.w, d.x_row = a.x_row, d.w_row = a.w_row, d.w_group = a.w_group;
    d.x_rows = a.x_rows, d.y_rows = a.y_rows, d.y_row = a.y_row, d.bias = a.bias, d.y = a.y;
    d.start = a.start, d.x_place = a.x_place, d.y_place = a.y_place, d.fault = a.fault, d.x_div = a.x_div;
    d.entries = a.entries, d.groups = a.groups, d.inputs = a.inputs, d.outputs = a.outputs, d.gate = a.gate;
    d.y_vec = (uintptr_t)a.y % 8 == 0 && a.y_row % 4 == 0;
    d.splits = p.splits, d.k_split = p.k_split;
    d.tiles = (int)row_tiles(a.entries, a.groups, p.M);
    d.tiles_n = p.kernel == kFew ? (int)ceil_div(a.outputs, p.N) : (int)(p.blocks / d.tiles);
    return a.type == KK_BF16 ? expert_run<KK_BF16>(d, p, s) : expert_run<KK_F16>(d, p, s);
}

template <int T, int OUT>
static hipError_t adapter_run(ProductDev& d, const ProductPlan& p, hipStream_t s) {
    hipError_t rc = hipSuccess;
    if (d.adapters) {
        d.slots = d.entries <= 256 ? 16 : 2;
        rc = run_shrink<T>(d, s);
    }
    if (rc != hipSuccess) return rc;
    if (!p.joined) return d.adapters ? run_tiled<T, false, true, OUT>(d, p, s) : run_tiled<T, false, false, OUT>(d, p, s);
    rc = run_tiled<T, false, false, 0>(d, p, s);
    if (rc != hipSuccess) return rc;
    d.tiles_n = (int)ceil_div(d.outputs, 1024);
    return launch(expand_kernel<T, OUT>, dim3((unsigned)((int64_t)d.entries * d.tiles_n)), dim3(256), 0, s, d);
}

hipError_t launch_adapter_product(const kk_adapter_product_args& a, const ProductPlan& p, hipStream_t s) {
    ProductDev d{};
    d.x = (const uint16_t*)a.x, d.w = (const uint16_t*)a.w, d.x_row = a.x_row, d.w_row = a.w_row;
    d.x_rows = d.y_rows = a.rows, d.y_row = a.y_row, d.bias = a.bias, d.y = a.y, d.fault = a.fault;
    d.entries = a.rows, d.groups = 1, d.inputs = a.inputs, d.outputs = a.outputs;
    const int e = a.out_type == KK_F32 ? 4 : 2;
    d.y_vec = (uintptr_t)a.y % (4 * e) == 0 && a.y_row % 4 == 0;
    d.splits = p.splits, d.k_split = p.k_split;
    d.tiles = (int)ceil_div(a.rows, p.M), d.tiles_n = (int)ceil_div(a.outputs, p.N);
    d.adapters = a.adapters;
    if (a.adapters) {
        d.a = (const uint16_t*)a.a, d.b = (const uint16_t*)a.b, d.scale = a.scale, d.adapter = a.adapter, d.rank = a.rank;
        char* ws = (char*)a.workspace;
        if (p.joined)
            d.h = (float*)(ws + p.ws_h);
        else
            d.h2 = (uint16_t*)(ws + p.ws_h), d.h_unit = (float*)(ws + p.ws_unit);
    }
    d.part = (float*)((char*)a.workspace + p.ws_part);
    if (a.type == KK_BF16) return a.out_type == KK_F32 ? adapter_run<KK_BF16, KK_F32>(d, p, s) : adapter_run<KK_BF16, KK_BF16>(d, p, s);
    return a.out_type == KK_F32 ? adapter_run<KK_F16, KK_F32>(d, p, s) : adapter_run<KK_F16, KK_F16>(d, p, s);
}

}  // namespace kk
