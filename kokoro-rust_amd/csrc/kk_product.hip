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

// Every lane of a wave calls this; false where the tile is empty.  `report`: this wave tells of bad groups.
template <int M>
__device__ __forceinline__ bool find_rows(const ProductDev& p, int tile, bool report, Rows& r) {
    if (!p.start) return group_rows(0, p.entries, 0, tile, M, r);
    const int lane = threadIdx.x & 63;
    bool found = false;
    for (int g0 = 0; g0 < p.groups; g0 += 256) {
        int s0[4], s1[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int g = min(g0 + 64 * j + lane, p.groups - 1);
            s0[j] = p.start[g], s1[j] = p.start[g + 1];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int g = g0 + 64 * j + lane;
            int i;
            const bool ok = group_ok(s0[j], s1[j], p.entries);
            if (report && g < p.groups && !ok) fault(p, KK_PRODUCT_BAD_START);
            const uint64_t who = __ballot(g < p.groups && ok && group_has(s0[j], s1[j], g, tile, M, i));
            if (found || !who) continue;
            const int at = __ffsll((unsigned long long)who) - 1;
            i = __builtin_amdgcn_readlane(i, at);
            found = group_rows(__builtin_amdgcn_readlane(s0[j], at), __builtin_amdgcn_readlane(s1[j], at), g0 + 64 * j + at, i, M, r);
        }
        if (found && !report) break;
    }
    return found;
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

// Up to 16 NT rows of a group and 16 MT rows of its matrix (8 MT gates and their partners) a unit.  Bound by reading the matrix once:
// nothing goes through LDS on its way in, a lane's 16-byte loads are the MFMA operands, and the next J steps of 32 inputs are under way
// while these ones' products run.  A unit's inputs are shared by KS waves, so that there are waves enough
// to cover the memory's latency also where there are few units; they leave their sums in LDS, and the block's threads join them.
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves;

// acc of the inputs that wave ks of KS takes.
template <int T, int MT, int NT, int KS>
__device__ __forceinline__ void few_sums(const uint16_t* const (&w)[MT], const uint16_t* const (&x)[NT], int inputs, int ks, f32x4 (&acc)[MT][NT]) {
    constexpr int kBest = (MT * NT >= 8 ? 20 : 10) / (MT + NT), J = kBest > 1 ? kBest : 1, kTurn = 32 * J;  // what registers hold
    const int at = ((threadIdx.x & 63) >> 4) * 8;
    uint4 a[2][J][MT], b[2][J][NT];
    const int per = (int)(ceil_div(inputs, 64 * KS) * 64), end = min(inputs, (ks + 1) * per);
    auto load = [&](int set, int k0) {
        if (k0 + kTurn <= end) {
#pragma unroll
            for (int j = 0; j < J; j++) {
#pragma unroll
                for (int t = 0; t < MT; t++) a[set][j][t] = stream_load((const uint4*)(w[t] + k0 + j * 32 + at));
#pragma unroll
                for (int n = 0; n < NT; n++) b[set][j][n] = *(const uint4*)(x[n] + k0 + j * 32 + at);
            }
        } else {
            const uint4 zero = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int k = k0 + j * 32 + at;
                const bool in = k < end;
#pragma unroll
                for (int t = 0; t < MT; t++) a[set][j][t] = in ? *(const uint4*)(w[t] + k) : zero;
#pragma unroll
                for (int n = 0; n < NT; n++) b[set][j][n] = in ? *(const uint4*)(x[n] + k) : zero;
            }
        }
    };
    auto mul = [&](int set) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int n = 0; n < NT; n++) acc[t][n] = Mat<T>::mul(a[set][j][t], b[set][j][n], acc[t][n]);
    };
    int k = ks * per;
    if (k >= end) return;
    load(0, k);
    for (; k + kTurn < end; k += 2 * kTurn) {
        load(1, k + kTurn);
        mul(0);
        if (k + 2 * kTurn < end) load(0, k + 2 * kTurn);
        mul(1);
    }
    if (k < end) mul(0);
}

// h = s a x of 16 rows and 32 ranks.  A block takes every slots-th of the adapters that its rows have.
template <int T>
__device__ __forceinline__ void few_shrink(const ProductDev& p, int block, float* lds) {
    constexpr int kLd = 36;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int slot = block % p.slots, ranks = (p.rank + 31) / 32, rest = block / p.slots;
    const int r0 = rest % ranks * 32, first = rest / ranks * 16, count = min(16, p.entries - first);
    const int own = col < count ? adapter_of(p, first + col) : -1;
    const uint16_t* const x[1] = {p.x + (int64_t)(first + min(col, count - 1)) * p.x_row};
    int id = -1;
    for (int n = 0;; n++) {
        int m = own > id ? own : INT32_MAX;
#pragma unroll
        for (int d = 8; d; d >>= 1) m = min(m, __shfl_xor(m, d));
        id = __builtin_amdgcn_readfirstlane(m);
        if (id == INT32_MAX) return;
        if (n % p.slots != slot) continue;
        const uint16_t* w[2];
        f32x4 acc[2][1] = {};
#pragma unroll
        for (int t = 0; t < 2; t++) w[t] = p.a + ((int64_t)id * p.rank + min(r0 + t * 16 + col, p.rank - 1)) * p.inputs;
        few_sums<T, 2, 1, kFewWaves>(w, x, p.inputs, wave, acc);
        __syncthreads();  // the sums of the adapter before have been read
#pragma unroll
        for (int t = 0; t < 2; t++) *(f32x4*)&lds[(wave * 16 + col) * kLd + t * 16 + g * 4] = acc[t][0];
        __syncthreads();
        const int row = threadIdx.x >> 5, k = threadIdx.x & 31;
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < kFewWaves; j++) v += lds[(j * 16 + row) * kLd + k];
        if (__shfl(own, row) == id && r0 + k < p.rank) p.h[(int64_t)(first + row) * p.rank + r0 + k] = v * p.scale[id];
    }
}

// OUT = 0: sums to `part`, and the first p.shrink blocks work on the adapters meanwhile.
template <int T, int MT, int NT, int KS, bool GATED, int OUT>
__global__ void __launch_bounds__(kFewThreads, NT * MT >= 8 ? 2 : 4) few_kernel(ProductDev p) {
    constexpr int N = 16 * MT, kOut = GATED ? N / 2 : N, kUnits = kFewWaves / KS, kLd = N + 4;
    constexpr int kSums = KS > 1 ? kFewWaves * 16 * NT * kLd : 4;
    __shared__ __align__(16) float lds[OUT == 0 && kSums < kFewWaves * 16 * 36 ? kFewWaves * 16 * 36 : kSums];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4, unit = wave / KS, ks = wave % KS;
    int block = blockIdx.x;
    if constexpr (OUT == 0) {
        if (block < p.shrink) {
            few_shrink<T>(p, block, lds);
            return;
        }
        block -= p.shrink;
    }
    const int tile = block / p.tiles_n, n0 = (block % p.tiles_n * kUnits + unit) * kOut;
    Rows r;
    if (!find_rows<16 * NT>(p, tile, blockIdx.x == 0 && wave == 0, r)) return;
    f32x4 acc[MT][NT] = {};
    if (n0 < p.outputs) {
        const uint16_t* wg = p.w + r.g * p.w_group;
        const uint16_t *w[MT], *x[NT];
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const int part = GATED ? t & 1 : 0, o = min(n0 + (GATED ? t >> 1 : t) * 16 + col, p.outputs - 1);
            w[t] = wg + (int64_t)(part * p.outputs + o) * p.w_row;
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int64_t from = x_of(p, r.first + min(n * 16 + col, r.count - 1));
            x[n] = p.x + max(from, (int64_t)0) * p.x_row;
        }
        few_sums<T, MT, NT, KS>(w, x, p.inputs, ks, acc);
    }
    const float* bias = p.bias ? p.bias + (int64_t)r.g * p.outputs * (GATED ? 2 : 1) : nullptr;
    // four outputs from n0 + o on of row `row` of the tile
    auto finish = [&](int row, int n0, int o, f32x4 v, f32x4 z) {
        const int left = p.outputs - (n0 + o), e = r.first + row;
        if (left <= 0) return;
        if constexpr (OUT == 0) {
            const float f[4] = {v[0], v[1], v[2], v[3]};
            store4<KK_F32>(p.part, (int64_t)e * p.outputs + n0 + o, p.outputs % 4 == 0, left, f);
        } else {
            const int64_t to = y_of(p, e);
            if (to < 0 || (p.x_place && x_of(p, e) < 0)) return;
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = n0 + o + min(i, left - 1);
                f[i] = bias ? v[i] + bias[at] : v[i];
                if constexpr (GATED) f[i] = gated(p.gate, f[i], bias ? z[i] + bias[p.outputs + at] : z[i]);
            }
            store4<OUT>(p.y, to * p.y_row + n0 + o, p.y_vec, left, f);
        }
    };
    if constexpr (KS == 1) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (n * 16 + col >= r.count) continue;
#pragma unroll
            for (int t = 0; t < MT; t += GATED ? 2 : 1) finish(n * 16 + col, n0, t * (GATED ? 8 : 16) + g * 4, acc[t][n], acc[GATED ? t + 1 : t][n]);
        }
    } else {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < MT; t++) *(f32x4*)&lds[((wave * NT + n) * 16 + col) * kLd + t * 16 + g * 4] = acc[t][n];
        __syncthreads();
        const int per = kUnits * (kOut / 4);
        for (int t = threadIdx.x; t < r.count * per; t += kFewThreads) {
            const int row = t / per, u = t % per / (kOut / 4), o = t % (kOut / 4) * 4;
            auto total = [&](int n) {
                f32x4 v = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KS; i++) v += *(const f32x4*)&lds[((u * KS + i) * 16 * NT + row) * kLd + n];
                return v;
            };
            const int at = GATED ? o / 16 * 32 + o % 16 : o;
            finish(row, (block % p.tiles_n * kUnits + u) * kOut, o, total(at), total(GATED ? at + 16 : at));
        }
    }
}

// ------------------------------------------------------------------ many rows

// Memory to LDS, 16 bytes a lane, in the lanes' order from `to` on (which is the wave's).  Written out because the compiler waits for
// all such loads before any read of LDS behind one; the waits here are counted by hand.  It has no output register.
__device__ __forceinline__ uint32_t lds_at(const uint16_t* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}
__device__ __forceinline__ void to_lds(const uint16_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
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
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wm = wave / WN;
    // blocks go to the 8 XCDs in turn: an XCD takes tiles that follow each other, which share rows of x and matrices in its L2
    const int per = gridDim.x / 8, t = blockIdx.x % 8 * per + blockIdx.x / 8;
    // eight tiles' width of outputs at a time
    const int all = p.tiles * p.splits, strip = t / (8 * all), wide = min(8, p.tiles_n - 8 * strip), in_strip = t - strip * 8 * all;
    if (wide <= 0) return;
    const int n0 = (8 * strip + in_strip % wide) * kOutN, rest = in_strip / wide;
    const int split = rest % p.splits, tile = rest / p.splits;
    Rows r;
    if (tile >= p.tiles || !find_rows<BM>(p, tile, blockIdx.x == 0 && wave == 0, r)) return;

    const int in_load = lane / kPieces;
    const int piece = (lane % kPieces) ^ (BK == 64 ? (in_load >> 1) + 4 * (wave & 1) : in_load >> 2);  // which one the lane loads
    const int k_lo = split * p.k_split, k_hi = min(p.inputs, k_lo + p.k_split);
    const uint16_t* wg = p.w + r.g * p.w_group + k_lo;
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
        src[QW + q] = p.x + max(from, (int64_t)0) * p.x_row + k_lo + piece * 8;
    }
    const int rest_k = (k_hi - k_lo) % BK, steps = (k_hi - k_lo) / BK;

    f32x16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int k = 0; k < 16; k++) acc[i][j][k] = 0.0f;
    uint4 fa[2][FN], fb[2][FM];
    const int col = lane & 31, half = lane >> 5, turn = BK == 64 ? (col >> 1) & 7 : (col >> 2) & 3;
    // operand i of sub-step kk: the matrix's tiles, then the rows'
    auto read = [&](int set, const uint16_t* stage, int kk, int i) {
        const int at = ((kk * 2 + half) ^ turn) * 8;
        if (i < FN)
            fa[set][i] = *(const uint4*)(stage + (wn * (BN / WN) + i * 32 + col) * BK + at);
        else
            fb[set][i - FN] = *(const uint4*)(stage + (BN + wm * (BM / WM) + (i - FN) * 32 + col) * BK + at);
    };
    uint16_t* const mine_in = lds + wave * (kRowsIn * BK);  // where this wave's first load of a stage goes
    const uint32_t in_at = lds_at(mine_in);
    auto load = [&](int q, int side) { to_lds(src[q], in_at + side * (2 * kStage) + q * (2 * kWaves * kRowsIn * BK)); };
    auto barrier = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // the first whole steps are on their way while the others, through the last buffer, run
#pragma unroll
    for (int i = 0; i < S - 1; i++)
        if (i < steps) {
#pragma unroll
            for (int q = 0; q < Q; q++) {
                load(q, i);
                src[q] += i + 1 < steps ? BK : 0;
            }
        }

    auto slow_step = [&](auto&& fill) {
        barrier();  // its buffer has been read
        fill(mine_in + (S - 1) * kStage);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        barrier();
#pragma unroll
        for (int kk = 0; kk < kSub; kk++) {
#pragma unroll
            for (int i = 0; i < FN + FM; i++) read(0, lds + (S - 1) * kStage, kk, i);
#pragma unroll
            for (int m = 0; m < FN * FM; m++)
                acc[m % FN][m / FN] = Mat<T>::mul(fa[0][m % FN], fb[0][m / FN], acc[m % FN][m / FN]);
        }
    };
    const uint4 zero = {0, 0, 0, 0};
    if constexpr (EXT) {
        // the adapters of the tile's rows, as more inputs: each one's b beside the rows' h, which is zero in rows of another
        constexpr int kIds = (BM + 63) / 64;
        int ids[kIds], mine[QX];  // of the tile's rows, a lane each; and of the rows that this lane loads
#pragma unroll
        for (int i = 0; i < kIds; i++) ids[i] = i * 64 + lane < r.count ? adapter_of(p, r.first + i * 64 + lane) : -1;
#pragma unroll
        for (int q = 0; q < QX; q++) {
            const int row = (q * kWaves + wave) * kRowsIn + in_load;
            mine[q] = row < r.count ? adapter_of(p, r.first + row) : -1;
        }
        bool any = false;
        for (int id = -1;;) {
            int m = INT32_MAX;
#pragma unroll
            for (int i = 0; i < kIds; i++)
                if (ids[i] > id) m = min(m, ids[i]);
#pragma unroll
            for (int d = 32; d; d >>= 1) m = min(m, __shfl_xor(m, d));
            id = __builtin_amdgcn_readfirstlane(m);
            if (id == INT32_MAX) break;
            any = true;
            for (int k0 = 0; k0 < 2 * p.rank; k0 += BK)
                slow_step([&](uint16_t* to) {
                    const int at = k0 + piece * 8;  // of a row of h2, whose b lies at half of it
                    const bool in = at < 2 * p.rank;
#pragma unroll
                    for (int q = 0; q < QW; q++) {
                        const int o = min(n0 + (q * kWaves + wave) * kRowsIn + in_load, p.outputs - 1);
                        uint16_t* dst = to + q * kWaves * kRowsIn * BK;
                        if (in)
                            to_lds(p.b + ((int64_t)id * p.outputs + o) * p.rank + at / 16 * 8, lds_at(dst));
                        else
                            *(uint4*)(dst + lane * 8) = zero;
                    }
#pragma unroll
                    for (int q = 0; q < QX; q++) {
                        const int row = min((q * kWaves + wave) * kRowsIn + in_load, r.count - 1);
                        uint16_t* dst = to + (QW + q) * kWaves * kRowsIn * BK;
                        if (in && mine[q] == id)
                            to_lds(p.h2 + (int64_t)(r.first + row) * (2 * p.rank) + at, lds_at(dst));
                        else
                            *(uint4*)(dst + lane * 8) = zero;
                    }
                });
        }
        if (T == KK_F16 && any) {
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
    }
    if (rest_k)  // the inputs behind the last whole step
        slow_step([&](uint16_t* to) {
            const int ahead = max(min(S - 1, steps - 1), 0) * BK;  // what src has been moved on by
#pragma unroll
            for (int q = 0; q < Q; q++) {
                uint16_t* dst = to + q * kWaves * kRowsIn * BK;
                if (piece * 8 < rest_k)
                    to_lds(src[q] + (steps * BK - ahead), lds_at(dst));
                else
                    *(uint4*)(dst + lane * 8) = zero;
            }
        });

    if (steps) {
        // all but the last S - 2 stages' loads of this wave have arrived, and then of all
        auto wait = [&] {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * Q) : "memory");
            barrier();
        };
        if (S - 1 > steps)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        wait();
#pragma unroll
        for (int i = 0; i < FN + FM; i++) read(0, lds, 0, i);
        int side = 0, into = S - 1;
        for (int i = 0; i < steps; i++) {
            const uint16_t* stage = lds + side * kStage;
            side = side + 1 == S ? 0 : side + 1;
            // behind the last step its loads are made once more, which keeps the count of those in flight; nothing reads them
            const int step = i + S < steps ? BK : 0;
#pragma unroll
            for (int kk = 0; kk < kSub; kk++) {
                const bool last = kk == kSub - 1;
                if (last) {
                    wait();
                    stage = lds + side * kStage;
                }
                constexpr int kLoadSubs = kSub > 2 ? kSub / 2 : 1;
                int next = 0, q = kk * Q / kLoadSubs;
                const int q_end = kk < kLoadSubs ? (kk + 1) * Q / kLoadSubs : q;
#pragma unroll
                for (int m = 0; m < FN * FM; m++) {
                    acc[m % FN][m / FN] = Mat<T>::mul(fa[kk & 1][m % FN], fb[kk & 1][m / FN], acc[m % FN][m / FN]);
#pragma unroll
                    for (; next * (FN * FM) < (m + 1) * (FN + FM); next++)
                        if (next < FN + FM) read(~kk & 1, stage, last ? 0 : kk + 1, next);
#pragma unroll
                    for (int n = 0; n < (Q + FN * FM - 1) / (FN * FM) + 1; n++)
                        if (q < q_end && (q - kk * Q / kLoadSubs) * (FN * FM) < (m + 1) * (q_end - kk * Q / kLoadSubs)) {
                            load(q, into);
                            src[q] += step;
                            q++;
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            into = into + 1 == S ? 0 : into + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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

// The same for many rows, all ranks, as two parts of 16 bits each.
template <int T, int MT>
__global__ void __launch_bounds__(64 * kFewWaves) shrink_kernel(ProductDev p) {
    constexpr int kLd = 16 * MT + 4;
    __shared__ __align__(16) float sums[kFewWaves][16][kLd];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int slot = blockIdx.x % p.slots, first = blockIdx.x / p.slots * 16, count = min(16, p.entries - first);
    const int own = col < count ? adapter_of(p, first + col) : -1;
    const uint16_t* const x[1] = {p.x + (int64_t)(first + min(col, count - 1)) * p.x_row};
    int id = -1;
    for (int n = 0;; n++) {
        int m = own > id ? own : INT32_MAX;
#pragma unroll
        for (int d = 8; d; d >>= 1) m = min(m, __shfl_xor(m, d));
        id = __builtin_amdgcn_readfirstlane(m);
        if (id == INT32_MAX) return;
        if (n % p.slots != slot) continue;
        const uint16_t* w[MT];
        f32x4 acc[MT][1] = {};
#pragma unroll
        for (int t = 0; t < MT; t++) w[t] = p.a + ((int64_t)id * p.rank + min(t * 16 + col, p.rank - 1)) * p.inputs;
        few_sums<T, MT, 1, kFewWaves>(w, x, p.inputs, wave, acc);
        __syncthreads();  // the sums of the adapter before have been read
#pragma unroll
        for (int t = 0; t < MT; t++) *(f32x4*)&sums[wave][col][t * 16 + g * 4] = acc[t][0];
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

template <int T>
__global__ void __launch_bounds__(kFewThreads) shrink_f32_kernel(ProductDev p) {
    __shared__ __align__(16) float lds[kFewWaves * 16 * 36];
    few_shrink<T>(p, blockIdx.x, lds);
}

// y = the sum of the parts + bias + b h.  A block takes one row and 1,024 outputs.
template <int T, int OUT>
__global__ void __launch_bounds__(256) expand_kernel(ProductDev p) {
    const int row = blockIdx.x / p.tiles_n, o = blockIdx.x % p.tiles_n * 1024 + threadIdx.x * 4, left = p.outputs - o;
    if (left <= 0) return;
    const int id = p.adapters ? adapter_of(p, row) : -1;
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
    if (p.bias)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] += p.bias[o + min(i, left - 1)];
    if (id >= 0) {
        const float* h = p.h + (int64_t)row * p.rank;
        const uint16_t* b[4];
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = p.b + ((int64_t)id * p.outputs + o + min(i, left - 1)) * p.rank;
        for (int k = 0; k < p.rank; k += 8) {
            uint16_t e[4][8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint4 q = *(const uint4*)(b[i] + k);
                __builtin_memcpy(e[i], &q, 16);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = h[k + j];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = fmaf(ElemOf<T>::load(e[i][j]), x, v[i]);
            }
        }
    }
    store4<OUT>(p.y, (int64_t)row * p.y_row + o, p.y_vec, left, v);
}

// ------------------------------------------------------------------ launches

template <int T, bool GATED, bool EXT, int OUT>
hipError_t run_tiled(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)((p.blocks + 7) / 8 * 8)), block(256);
    if (p.M == 256) return launch(tiled_kernel<T, 256, 256, 2, 4, 64, 2, 1, GATED, EXT, OUT>, grid, dim3(512), 0, s, d);
    if (p.M == 128) return launch(tiled_kernel<T, 128, 128, 2, 2, 64, 2, 2, GATED, EXT, OUT>, grid, block, 0, s, d);
    return launch(tiled_kernel<T, 128, 64, 2, 2, 64, 2, 2, GATED, EXT, OUT>, grid, block, 0, s, d);
}

template <int T, int MT, int NT, bool GATED, int OUT>
hipError_t run_few_ks(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.blocks + d.shrink)), block(kFewThreads);
    if (p.KS == 1) return launch(few_kernel<T, MT, NT, 1, GATED, OUT>, grid, block, 0, s, d);
    if (p.KS == 2) return launch(few_kernel<T, MT, NT, 2, GATED, OUT>, grid, block, 0, s, d);
    return launch(few_kernel<T, MT, NT, 8, GATED, OUT>, grid, block, 0, s, d);
}

template <int T, bool GATED, int OUT>
hipError_t run_few(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    constexpr int kTwo = GATED ? 2 : 1;
    if (p.M == 16 && p.N == 16) return run_few_ks<T, kTwo, 1, GATED, OUT>(d, p, s);
    if (p.M == 16) return run_few_ks<T, 2 * kTwo, 1, GATED, OUT>(d, p, s);
    if (p.M == 32) return run_few_ks<T, 2, 2, GATED, OUT>(d, p, s);
    if (p.M == 64) return run_few_ks<T, 2, 4, GATED, OUT>(d, p, s);
    return run_few_ks<T, 2, 6, GATED, OUT>(d, p, s);
}

template <int T>
hipError_t run_shrink(const ProductDev& d, hipStream_t s) {
    const dim3 grid((unsigned)(ceil_div(d.entries, 16) * d.slots)), block(kFewThreads);
    if (d.rank <= 16) return launch(shrink_kernel<T, 1>, grid, block, 0, s, d);
    if (d.rank <= 32) return launch(shrink_kernel<T, 2>, grid, block, 0, s, d);
    if (d.rank <= 64) return launch(shrink_kernel<T, 4>, grid, block, 0, s, d);
    if (d.rank <= 128) return launch(shrink_kernel<T, 8>, grid, block, 0, s, d);
    return launch(shrink_kernel<T, 16>, grid, block, 0, s, d);
}

}  // namespace

// Few rows: the rows a tile, outputs a unit, and waves that share a unit's inputs: 16 waves a CU where the units allow it.
// `tiles`: row tiles that are likely to hold rows.
static void few_plan(ProductPlan& p, int M, int64_t tiles, int64_t bound, int outputs, bool gate, int inputs, int n_cu) {
    p.kernel = kFew, p.M = M;
    const int64_t waves = (int64_t)n_cu * 16;
    // 32 outputs a unit (with gates 16, or 32): half the reads of x
    p.N = M == 16 ? (tiles * ceil_div(outputs, 32) >= waves / 8 ? 32 : 16) : gate ? 16 : 32;
    const int64_t units = tiles * ceil_div(outputs, p.N);
    p.KS = units >= waves ? 1 : units >= waves / 2 ? 2 : 8;
    p.blocks = bound * ceil_div(outputs, p.N * (kFewWaves / p.KS));
}

ProductPlan expert_plan(const kk_expert_product_args& a, int n_cu) {
    ProductPlan p{};
    p.splits = 1, p.k_split = a.inputs;
    const bool gate = a.gate != KK_GATE_NONE;
    const int64_t wide = (int64_t)a.outputs * (gate ? 2 : 1), mean = a.entries / a.groups;
    if (mean <= 48) {
        const int M = mean <= 12 ? 16 : mean <= 24 ? 32 : 64;
        few_plan(p, M, std::min<int64_t>(a.entries, a.groups), row_tiles(a.entries, a.groups, M), a.outputs, gate, a.inputs, n_cu);
        return p;
    }
    p.kernel = kTiled;
    p.M = mean >= 384 ? 256 : mean >= 96 ? 128 : 64;
    p.N = p.M == 256 ? 256 : 128;
    p.blocks = row_tiles(a.entries, a.groups, p.M) * ceil_div(wide, p.N);
    return p;
}

ProductPlan adapter_plan(const kk_adapter_product_args& a, int n_cu) {
    ProductPlan p{};
    p.splits = 1, p.k_split = a.inputs;
    auto tiles = [&](int M, int N) { return ceil_div(a.rows, M) * ceil_div(a.outputs, N); };
    if (a.rows <= 96) {
        const int M = a.rows <= 16 ? 16 : a.rows <= 32 ? 32 : a.rows <= 64 ? 64 : 96;
        few_plan(p, M, 1, 1, a.outputs, false, a.inputs, n_cu);
        p.joined = a.adapters > 0;
    } else {
        p.kernel = kTiled;
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
    d.tiles_n = (int)(p.blocks / d.tiles);
    return a.type == KK_BF16 ? expert_run<KK_BF16>(d, p, s) : expert_run<KK_F16>(d, p, s);
}

template <int T, int OUT>
static hipError_t adapter_run(ProductDev& d, const ProductPlan& p, hipStream_t s) {
    d.slots = d.entries <= 256 ? std::min(16, d.entries) : 2;
    hipError_t rc;
    if (p.kernel == kFew) {
        if (!p.joined) return run_few<T, false, OUT>(d, p, s);
        d.shrink = (int)(ceil_div(d.entries, 16) * ceil_div(d.rank, 32) * d.slots);
        rc = run_few<T, false, 0>(d, p, s);
    } else {
        if (d.adapters && p.joined)
            rc = launch(shrink_f32_kernel<T>, dim3((unsigned)(ceil_div(d.entries, 16) * ceil_div(d.rank, 32) * d.slots)), dim3(kFewThreads), 0, s, d);
        else
            rc = d.adapters ? run_shrink<T>(d, s) : hipSuccess;
        if (rc != hipSuccess) return rc;
        if (!p.joined) return d.adapters ? run_tiled<T, false, true, OUT>(d, p, s) : run_tiled<T, false, false, OUT>(d, p, s);
        rc = run_tiled<T, false, false, 0>(d, p, s);
    }
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
    d.tiles = (int)ceil_div(a.rows, p.M), d.tiles_n = (int)(p.blocks / p.splits / d.tiles);
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
