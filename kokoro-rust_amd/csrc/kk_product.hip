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

// The row of x that entry e's place means, or -1.
__device__ __forceinline__ int x_of(const ProductDev& p, int e, int place) {
    if (!p.x_place) return e;
    // place / x_div: the half keeps the product's rounding away from whole numbers
    const int row = (int)(((double)place + 0.5) * p.x_inv);
    if (place >= 0 && row < p.x_rows) return row;
    fault(p, KK_PRODUCT_BAD_PLACE);
    return -1;
}
// The row of y, or -1.
__device__ __forceinline__ int y_of(const ProductDev& p, int e, int place) {
    if (!p.y_place) return e;
    if (place >= 0 && place < p.y_rows) return place;
    fault(p, KK_PRODUCT_BAD_PLACE);
    return -1;
}
__device__ __forceinline__ int adapter_in(const ProductDev& p, int id) {
    if (id >= p.adapters) fault(p, KK_PRODUCT_BAD_ADAPTER);
    return id >= p.adapters || id < 0 ? -1 : id;
}
__device__ __forceinline__ int adapter_of(const ProductDev& p, int row) { return adapter_in(p, p.adapter[row]); }

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

// ------------------------------------------------------------------ a tile

// N rows of the matrix (outputs) and M rows of x, held by WN x WM waves in 32 x 32 tiles of the matrix cores, through LDS in S stages of
// K inputs each.
template <int N_, int M_, int WN_, int WM_, int K_, int S_, int PER_CU_>
struct Tile {
    static constexpr int N = N_, M = M_, WN = WN_, WM = WM_, K = K_, S = S_, kPerCu = PER_CU_;
    static constexpr int kWaves = WN * WM, kThreads = 64 * kWaves;
    static constexpr int FN = N / WN / 32, FM = M / WM / 32;
    static constexpr int kPieces = K / 8, kRowsIn = 64 / kPieces;  // of 16 bytes of a row, and rows that a wave's load covers
    static constexpr int QW = N / kRowsIn / kWaves, QX = M / kRowsIn / kWaves, Q = QW + QX;
    static constexpr int kStage = (N + M) * K;  // in values
    static constexpr int kNext = kWaves * kRowsIn * K;  // from a wave's load to its next in LDS
    static_assert(QW * kRowsIn * kWaves == N && QX * kRowsIn * kWaves == M && kWaves % 2 == 0, "tile");
};

// Memory to LDS, 16 bytes a lane, in the lanes' order from `to` on (which is the wave's).  Written out because the compiler waits for
// all such loads before any read of LDS behind one; the waits here are counted by hand.  It has no output register, and nothing
// else here uses m0.
__device__ __forceinline__ uint32_t lds_at(const uint16_t* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}
__device__ __forceinline__ void to_lds(const uint16_t* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(from) : "memory");
}
__device__ __forceinline__ void word_to_lds(const int32_t* from, uint32_t to) {  // 4 bytes a lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(from) : "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// What a wave and a lane are in a tile.  A stage's rows are 64 inputs, eight pieces of 16 bytes, in an order that their row number turns
// (by XOR with its bits 1 to 3; rows of 32 inputs, four pieces: bits 2 and 3), so that the 16 rows that LDS reads at once lie on all 64
// banks (with bits 0 to 2 half of its time were conflicts); since the loads store lane after lane, the order is made by which piece each
// lane loads.
template <class C>
struct Place {
    int lane, wave, wn, wm, col, half, row_in, piece;
    int a_row, b_row, turn;  // where this lane's operands lie in a stage
    uint16_t *lds, *in;  // `in`: where this wave's first load of a stage goes
    uint32_t in_at;
    __device__ __forceinline__ explicit Place(uint16_t* l) : lds(l) {
        lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wn = wave % C::WN, wm = wave / C::WN;
        col = lane & 31, half = lane >> 5, turn = half ^ (C::K == 64 ? (col >> 1) & 7 : (col >> 2) & 3);
        a_row = (wn * (C::N / C::WN) + col) * C::K, b_row = (C::N + wm * (C::M / C::WM) + col) * C::K;
        const int in_load = lane / C::kPieces;
        row_in = wave * C::kRowsIn + in_load;
        piece = ((lane % C::kPieces) ^ (C::K == 64 ? (in_load >> 1) + 4 * (wave & 1) : in_load >> 2)) * 8;
        in = lds + wave * (C::kRowsIn * C::K);
        in_at = lds_at(in);
    }
    __device__ __forceinline__ int row(int q) const { return q * (C::kWaves * C::kRowsIn) + row_in; }  // of this lane's load q
};

template <class C>
__device__ __forceinline__ void load(const Place<C>& at, const uint16_t* const (&src)[C::Q], int q, int side) {
    to_lds(src[q], at.in_at + side * (2 * C::kStage) + q * (2 * C::kNext));
}

// The first of `steps` stages' loads, as many as are in flight at a time.
template <class C>
__device__ __forceinline__ void begin(const Place<C>& at, const uint16_t* (&src)[C::Q], int steps) {
#pragma unroll
    for (int i = 0; i < C::S - 1; i++)
        if (i < steps) {
#pragma unroll
            for (int q = 0; q < C::Q; q++) {
                load<C>(at, src, q, i);
                src[q] += C::K;
            }
        }
}

template <int T, class C>
struct Acc {
    f32x16 sum[C::FN][C::FM];
    uint4 a[2][C::FN], b[2][C::FM];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < C::FN; i++)
#pragma unroll
            for (int j = 0; j < C::FM; j++)
#pragma unroll
                for (int k = 0; k < 16; k++) sum[i][j][k] = 0.0f;
    }
    // operand i of the 16 inputs kk of a stage: the matrix's tiles, then the rows'
    __device__ __forceinline__ void read(const Place<C>& at, int set, const uint16_t* stage, int kk, int i) {
        const uint16_t* from = stage + ((kk * 2) ^ at.turn) * 8;
        if (i < C::FN)
            a[set][i] = *(const uint4*)(from + at.a_row + i * 32 * C::K);
        else
            b[set][i - C::FN] = *(const uint4*)(from + at.b_row + (i - C::FN) * 32 * C::K);
    }
    __device__ __forceinline__ void mul(int set, int m) {
        sum[m % C::FN][m / C::FN] = Mat<T>::mul(a[set][m % C::FN], b[set][m / C::FN], sum[m % C::FN][m / C::FN]);
    }
};

// The whole stages, whose first S - 1 `begin` has asked for.  The operands of the next 16 inputs are read, and the loads of a later
// stage made, between the products of these; sched_barrier keeps that order.  A wave without rows only loads.
template <int T, class C>
__device__ __forceinline__ void run_stages(const Place<C>& place, const uint16_t* (&src)[C::Q], int steps, bool live, Acc<T, C>& acc) {
    constexpr int S = C::S, Q = C::Q, kMul = C::FN * C::FM, kRead = C::FN + C::FM, kSub = C::K / 16;
    if (!steps) return;
    // all but the last S - 2 stages' loads of this wave have arrived, and then of all; near the end there are fewer: all
    auto wait = [&](bool all) {
        if (all)
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * Q) : "memory");
        barrier();
    };
    wait(steps < S - 1);
    // whatever the addresses still depend on (a place's load, a register kept in scratch) is waited for here: a wait of the compiler's
    // own inside the loop would be for all loads
    Place<C> at = place;
    asm volatile("" : "+v"(at.a_row), "+v"(at.b_row), "+v"(at.turn));
#pragma unroll
    for (int q = 0; q < Q; q++) asm volatile("" : "+v"(src[q]));
    if (live) {
#pragma unroll
        for (int i = 0; i < kRead; i++) acc.read(at, 0, at.lds, 0, i);
    }
    int side = 0, into = S - 1;
    auto stage = [&](auto more, auto on, bool last_wait) {
        constexpr bool kMore = decltype(more)::value, kOn = decltype(on)::value;
        const uint16_t* from = at.lds + side * C::kStage;
        side = side + 1 == S ? 0 : side + 1;
#pragma unroll
        for (int kk = 0; kk < kSub; kk++) {
            const bool last = kk == kSub - 1;
            if (last) {
                wait(last_wait);
                from = at.lds + side * C::kStage;
            }
            // loads in the first half, so that they have the other to arrive
            constexpr int kIn = kSub > 2 ? kSub / 2 : 1;
            const int q0 = min(kk, kIn) * Q / kIn, q1 = min(kk + 1, kIn) * Q / kIn;
            if constexpr (kOn) {
                int next = 0, q = q0;
#pragma unroll
                for (int m = 0; m < kMul; m++) {
                    acc.mul(kk & 1, m);
#pragma unroll
                    for (int n = 0; n < kRead; n++)
                        if (next < kRead && next * kMul < (m + 1) * kRead) acc.read(at, ~kk & 1, from, last ? 0 : kk + 1, next), next++;
                    if constexpr (kMore)
#pragma unroll
                        for (int n = 0; n < Q; n++)
                            if (q < q1 && (q - q0) * kMul < (m + 1) * (q1 - q0)) {
                                load<C>(at, src, q, into);
                                src[q] += C::K;
                                q++;
                            }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else if constexpr (kMore) {
#pragma unroll
                for (int q = 0; q < Q; q++)
                    if (q >= q0 && q < q1) {
                        load<C>(at, src, q, into);
                        src[q] += C::K;
                    }
            }
        }
        into = into + 1 == S ? 0 : into + 1;
    };
    const int more = steps - (S - 1);
    // behind the last stage, what is read once more is what its buffer holds, and is not used
    if (live) {
        for (int i = 0; i < more; i++) stage(std::true_type(), std::true_type(), false);
        for (int i = max(more, 0); i < steps; i++) stage(std::false_type(), std::true_type(), true);
    } else {
        for (int i = 0; i < more; i++) stage(std::true_type(), std::false_type(), false);
        for (int i = max(more, 0); i < steps; i++) stage(std::false_type(), std::false_type(), true);
    }
}

// One stage through the last buffer that `fill(q, where)` loads or stores piece by piece, all waves together.
template <int T, class C, class F>
__device__ __forceinline__ void run_alone(const Place<C>& at, Acc<T, C>& acc, F&& fill) {
    barrier();  // the buffer has been read
    uint16_t* to = at.in + (C::S - 1) * C::kStage;
#pragma unroll
    for (int q = 0; q < C::Q; q++) fill(q, to + q * C::kNext);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    barrier();
#pragma unroll
    for (int kk = 0; kk < C::K / 16; kk++) {
#pragma unroll
        for (int i = 0; i < C::FN + C::FM; i++) acc.read(at, 0, at.lds + (C::S - 1) * C::kStage, kk, i);
#pragma unroll
        for (int m = 0; m < C::FN * C::FM; m++) acc.mul(0, m);
    }
}
template <class C>
__device__ __forceinline__ void piece_or_zero(const Place<C>& at, bool in, const uint16_t* from, uint16_t* to) {
    const uint4 zero = {0, 0, 0, 0};
    if (in)
        to_lds(from, lds_at(to));
    else
        *(uint4*)(to + at.lane * 8) = zero;
}

// The next adapter after `id` among the tile's rows, or INT32_MAX; ids: one row a lane.
template <int N>
__device__ __forceinline__ int next_adapter(const int (&ids)[N], int id) {
    int m = INT32_MAX;
#pragma unroll
    for (int i = 0; i < N; i++)
        if (ids[i] > id) m = min(m, ids[i]);
#pragma unroll
    for (int d = 32; d; d >>= 1) m = min(m, __shfl_xor(m, d));
    return __builtin_amdgcn_readfirstlane(m);
}

// ------------------------------------------------------------------ adapters: h = s a x

// Of 16 rows, 32 ranks and a share of the inputs, of every slots-th of the rows' adapters.  Straight from memory to registers, in 16-byte
// loads that are the operands; the waves share the inputs and leave their sums in LDS.  W * 16 * 36 floats of LDS.
// They run beside the main product's blocks, so that a's bytes are read while w's are: one row of 4,096 x 4,096 with rank 16 takes 9 us
// in one launch, 96 rows with 40 adapters of rank 32 21.
template <int T, int W>
__device__ __forceinline__ void shrink_few(const ProductDev& p, int block, float* lds) {
    constexpr int kLd = 36, J = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int split = block % p.h_splits, ranks = (p.rank + 31) / 32;
    int rest = block / p.h_splits;
    const int r0 = rest % ranks * 32;
    rest /= ranks;
    const int tiles = (p.entries + 15) / 16, slot = rest / tiles, first = rest % tiles * 16, count = min(16, p.entries - first);
    const int ids[1] = {col < count ? adapter_of(p, first + col) : -1};
    const int share = (p.h_k / W + 31) / 32 * 32;  // of a wave
    const int k_lo = split * p.h_k + wave * share, k_hi = min(min(p.inputs, (split + 1) * p.h_k), k_lo + share);
    const uint16_t* x = p.x + (int64_t)(first + max(min(col, count - 1), 0)) * p.x_row + g * 8;
    int id = -1;
    for (int n = 0;; n++) {
        id = next_adapter(ids, id);
        if (id == INT32_MAX) return;
        if (n % p.slots != slot) continue;
        const uint16_t* w[2];
        f32x4 acc[2] = {};
#pragma unroll
        for (int t = 0; t < 2; t++) w[t] = p.a + ((int64_t)id * p.rank + min(r0 + t * 16 + col, p.rank - 1)) * p.inputs + g * 8;
        for (int k0 = k_lo; k0 < k_hi; k0 += 32 * J) {
            const uint4 zero = {0, 0, 0, 0};
            uint4 a[J][2], b[J];
#pragma unroll
            for (int j = 0; j < J; j++) {
                const int k = k0 + 32 * j;
                const bool in = k + g * 8 < k_hi;
                b[j] = in ? *(const uint4*)(x + k) : zero;
#pragma unroll
                for (int t = 0; t < 2; t++) a[j][t] = in ? *(const uint4*)(w[t] + k) : zero;
            }
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int t = 0; t < 2; t++) acc[t] = Mat<T>::mul(a[j][t], b[j], acc[t]);
        }
        __syncthreads();  // the sums of the adapter before have been read
#pragma unroll
        for (int t = 0; t < 2; t++) *(f32x4*)&lds[(wave * 16 + col) * kLd + t * 16 + g * 4] = acc[t];
        __syncthreads();
        for (int i = threadIdx.x; i < 512; i += 64 * W) {
            const int row = i >> 5, k = i & 31;
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < W; j++) v += lds[(j * 16 + row) * kLd + k];
            if (__shfl(ids[0], row) == id && r0 + k < p.rank) p.h[((int64_t)split * p.entries + first + row) * p.rank + r0 + k] = v * p.scale[id];
        }
    }
}

// Of many rows: of a row tile, of every slots-th of its adapters, as tiles of the products are.  12,661 rows of 4,096 inputs and rank 64
// 36-38 us in 990 blocks (99 row tiles, two blocks for the adapters of each, the inputs in five parts): x (104 MB) is read once for all ranks up to
// 64, at 2.8 TB/s; the parts' sums (16 MB) are written here and added up by halves_kernel.
template <int T, class C>
__global__ void __launch_bounds__(C::kThreads, C::kPerCu * C::kWaves / 4) shrink_kernel(ProductDev p) {
    constexpr int K = C::K;
    __shared__ __align__(16) uint16_t lds[C::S * C::kStage];
    const Place<C> at(lds);
    Acc<T, C> acc;
    constexpr int kIds = (C::M + 63) / 64;
    const int n_ranks = (p.rank + C::N - 1) / C::N;
    int rest = blockIdx.x;
    const int split = rest % p.h_splits;
    rest /= p.h_splits;
    const int n0 = rest % n_ranks * C::N;
    rest /= n_ranks;
    const int tiles = (p.entries + C::M - 1) / C::M, slot = rest / tiles, first = rest % tiles * C::M;
    const int count = min(C::M, p.entries - first);
    int ids[kIds];
#pragma unroll
    for (int i = 0; i < kIds; i++) ids[i] = i * 64 + at.lane < count ? adapter_of(p, first + i * 64 + at.lane) : -1;
    const int k_lo = split * p.h_k, k_hi = min(p.inputs, k_lo + p.h_k), steps = (k_hi - k_lo) / K, left = (k_hi - k_lo) % K;
    int id = -1;
    for (int n = 0;; n++) {
        id = next_adapter(ids, id);
        if (id == INT32_MAX) return;
        if (n % p.slots != slot) continue;
        const uint16_t* src[C::Q];
#pragma unroll
        for (int q = 0; q < C::QW; q++)
            src[q] = p.a + ((int64_t)id * p.rank + min(n0 + at.row(q), p.rank - 1)) * p.inputs + k_lo + at.piece;
#pragma unroll
        for (int q = 0; q < C::QX; q++)
            src[C::QW + q] = p.x + (int64_t)(first + min(at.row(q), count - 1)) * p.x_row + k_lo + at.piece;
        acc.clear();
        barrier();  // an adapter before has been read
        begin<C>(at, src, steps);
        if (left)
            run_alone<T, C>(at, acc, [&](int q, uint16_t* to) {
                piece_or_zero(at, at.piece < left, src[q] + (steps - min(C::S - 1, steps)) * K, to);
            });
        run_stages<T, C>(at, src, steps, at.wm * (C::M / C::WM) < count && n0 + at.wn * (C::N / C::WN) < p.rank, acc);
        const float s = p.scale[id];
#pragma unroll
        for (int j = 0; j < C::FM; j++) {
            const int row = at.wm * (C::M / C::WM) + j * 32 + at.col;
            if (row >= count || adapter_of(p, first + row) != id) continue;
            float* to = p.h + ((int64_t)split * p.entries + first + row) * p.rank;
#pragma unroll
            for (int i = 0; i < C::FN; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int o = n0 + at.wn * (C::N / C::WN) + i * 32 + q * 8 + at.half * 4;
                    if (o >= p.rank) continue;  // a multiple of 8
                    const f32x4 v = {acc.sum[i][j][4 * q] * s, acc.sum[i][j][4 * q + 1] * s, acc.sum[i][j][4 * q + 2] * s,
                                     acc.sum[i][j][4 * q + 3] * s};
                    *(f32x4*)(to + o) = v;
                }
        }
    }
}

// ------------------------------------------------------------------ the products

// The groups' tiles summed up, in LDS: sums[g] of the groups before g, and starts[g].  The block's first wave makes it.  Beside more than some 890
// groups' eight bytes each, one block of 128 x 64 tiles fits a CU in place of two.
struct Groups {
    const int *sums, *starts;
    int tiles;
};
template <int M>
__device__ __forceinline__ Groups sum_groups(const ProductDev& p, int* lds) {
    if (!p.start) return {nullptr, nullptr, p.tiles};
    int *sums = lds, *starts = lds + p.groups + 1;
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int before = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 64) {
            const int g = g0 + lane, s0 = p.start[min(g, p.groups - 1)], s1 = p.start[min(g, p.groups - 1) + 1];
            const bool in = g < p.groups, ok = group_ok(s0, s1, p.entries);
            if (blockIdx.x == 0 && in && !ok) fault(p, KK_PRODUCT_BAD_START);
            const int own = in && ok ? (s1 - s0 + M - 1) / M : 0;
            int sum = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(sum, d);
                if (lane >= d) sum += y;
            }
            if (in) sums[g] = before + sum - own, starts[g] = s0;
            if (g == p.groups - 1) starts[g + 1] = s1, sums[g + 1] = before + sum;
            // groups that overlap could have more tiles than the launch was sized by: what is behind those is never asked for
            before = min(__builtin_amdgcn_readlane(before + sum, 63), p.tiles);
        }
    }
    __syncthreads();
    return {sums, starts, min(__builtin_amdgcn_readfirstlane(sums[p.groups]), p.tiles)};
}
template <int M>
__device__ __forceinline__ Rows rows_of(const ProductDev& p, const Groups& all, int tile) {
    Rows r;
    if (!p.start) {
        group_rows(0, p.entries, 0, tile, M, r);
        return r;
    }
    const int lane = threadIdx.x & 63;
    int g = p.groups - 1;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
        const uint64_t who = __ballot(all.sums[min(g0 + lane, p.groups - 1) + 1] > tile);
        if (!who) continue;
        g = min(g0 + __ffsll((unsigned long long)who) - 1, p.groups - 1);
        break;
    }
    const int s0 = __builtin_amdgcn_readfirstlane(all.starts[g]), s1 = __builtin_amdgcn_readfirstlane(all.starts[g + 1]);
    group_rows(s0, s1, g, tile - __builtin_amdgcn_readfirstlane(all.sums[g]), M, r);
    return r;
}

// Parts of 16 bits that h of many rows is kept in: of f16 (11 bits each) two; of bf16 (8) two, to 2^-17, where y has 16 bits, and three where it
// has 32: with two, f32 results were off by 1.1e-6 in place of 2.3e-7.
template <int T, int OUT>
constexpr int kHParts = T == KK_BF16 && OUT == KK_F32 ? 3 : 2;

// The adapters' shares in a wave's sums that are not finite once more, each row's from its own adapter's b and h as it was before it was split.
// Where h itself is NaN all of them are, and stay: rows of NaN cost nothing.  Every 128th output of all b infinite: 12,661 rows 451 -> 555 us.
template <int T, class C>
__device__ __forceinline__ void add_apart(const ProductDev& p, const Place<C>& at, const Rows& r, int n0, const int* adapters, Acc<T, C>& acc) {
#pragma unroll
    for (int j = 0; j < C::FM; j++) {
        const int in = at.wm * (C::M / C::WM) + j * 32 + at.col, row = r.first + min(in, r.count - 1);
        const int id = adapter_in(p, adapters[row - r.first]);
        if (in >= r.count || (id >= 0 && p.h_unit[row] != p.h_unit[row])) continue;
        const float* h = p.h + (int64_t)row * p.rank;
#pragma unroll
        for (int n = 0; n < 4 * C::FN; n++) {
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; e++) bad |= !(fabsf(acc.sum[n / 4][j][n % 4 * 4 + e]) < INFINITY);
            if (bad) {
                int o0 = n0 + n * 8 + at.half * 4;
                asm volatile("" : "+v"(o0));
                float sum[4] = {};
                for (int k0 = 0; id >= 0 && k0 < p.rank; k0 += 8) {
                    float v[8] = {};
                    for (int s = 0; s < p.h_splits; s++)
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] += h[(int64_t)s * p.h_rows * p.rank + k0 + k];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint16_t b[8];
                        const uint4 q = *(const uint4*)(p.b + ((int64_t)id * p.outputs + min(o0 + e, p.outputs - 1)) * p.rank + k0);
                        __builtin_memcpy(b, &q, 16);
                        float own = 0.0f;
#pragma unroll
                        for (int k = 0; k < 8; k++) own = fmaf(ElemOf<T>::load(b[k]), v[k], own);
                        sum[e] += own;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) acc.sum[n / 4][j][n % 4 * 4 + e] = sum[e];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// One product tile: rows of x, the outputs from n0 on, inputs from k_lo on.
struct Work {
    Rows r;
    int n0, split, k_lo, steps, rest;
};

// Bound by the matrix cores where a group has many rows, and then by the power they draw: 63,352 entries over 64 groups, 2,048 inputs to
// 2 x 1,024 outputs (531 GFLOP) 548-650 us by the device's clock, 820-970 TFLOP/s; one group of 8,192 x 8,192 x 8,192 1,200, of zeros 1,430
// (a library product 1,525 and 2,125).  11% of the tiles' rows are empty, 9 rounds of tiles are 8.7 full ones, and each tile costs 12 us beside
// its stages: the stores of all CUs come together and wait for memory (50 us of such a call).  Without its loads a stage of 64 inputs takes
// 1.5 us of 1.85, without its products 1.4.  Where groups have few rows, bound by the matrices' bytes: 512 entries over 64 groups of
// 2,048 x 1,024 (268 MB) 50 us, 5.4 TB/s; eight entries with a group each (67 MB) 14 us.
// Tried: four waves with 128 x 128 each (stages 7% shorter, tiles' ends 30% longer), five stages of 32 inputs and two of 64, loads spread
// over a whole stage or reads all in its first half (no change), blocks started apart in time so that their stores do not meet (no change),
// stores that pass the caches (a third slower), matrices straight to registers for few rows (15-20% slower: 64 bytes of each row a load).
// EXT: adapters in many rows, as more inputs (h2).  OUT = 0: sums to `part`, and the adapters' h in blocks behind p.blocks.
template <int T, class C, bool GATED, bool EXT, int OUT>
__global__ void __launch_bounds__(C::kThreads, C::kPerCu * C::kWaves / 4) product_kernel(ProductDev p) {
    constexpr int kOutN = GATED ? C::N / 2 : C::N, K = C::K;
    static_assert(!GATED || C::FN % 2 == 0, "a gate and its partner in one wave");
    __shared__ __align__(16) uint16_t lds[C::S * C::kStage];
    __shared__ __align__(16) int places[2][2][C::M];
    extern __shared__ int more_lds[];  // [2][groups + 1]
    const Place<C> at(lds);
    Acc<T, C> acc;

    if constexpr (OUT == 0) {
        // the adapters' blocks are the last: they run beside the others
        if ((int)blockIdx.x >= p.blocks) {
            shrink_few<T, C::kWaves>(p, blockIdx.x - p.blocks, (float*)lds);
            return;
        }
    }

    // a block takes tile after tile
    const Groups groups = sum_groups<C::M>(p, more_lds);
    const int tall = groups.tiles * p.splits;
    const TileWalk walk = tile_walk(blockIdx.x, p.blocks, tall * p.tiles_n);
    int t = walk.first;
    auto work_of = [&](int t) {
        Work w;
        const TileAt on = tile_at(t, tall, p.tiles_n);
        w.n0 = on.n * kOutN;
        const int rest = on.row;
        const int tile = rest / p.splits;
        w.split = rest - tile * p.splits;
        w.r = rows_of<C::M>(p, groups, tile);
        w.k_lo = w.split * p.k_split;
        const int k = min(p.inputs, w.k_lo + p.k_split) - w.k_lo;
        w.steps = k / K, w.rest = k % K;
        return w;
    };
    // Where a tile's rows of x and y are (EXT: its rows' adapters): loaded to LDS beside the tile before, so that nothing waits for a load
    // behind that tile's stores.
    auto ask = [&](const Work& w, int side) {
        const int32_t* const from[2] = {EXT ? p.adapter : p.x_place, p.y_place};
#pragma unroll
        for (int i = 0; i < 2 * C::M / 64; i += C::kWaves) {
            const int piece = i + at.wave, which = piece / (C::M / 64), r0 = piece % (C::M / 64) * 64;
            if (piece < 2 * C::M / 64 && from[which])
                word_to_lds(from[which] + w.r.first + min(r0 + at.lane, w.r.count - 1), lds_at((uint16_t*)&places[side][which][r0]));
        }
    };
    int to[C::FM];  // this lane's rows of y
    const uint16_t* src[C::Q];
    auto aim = [&](const Work& w, int side) {
        const uint16_t* wg = p.w + w.r.g * p.w_group + w.k_lo + at.piece;
#pragma unroll
        for (int q = 0; q < C::QW; q++) {
            const int row = at.row(q);
            int o;
            if constexpr (GATED)
                o = min(w.n0 + row / 64 * 32 + row % 32, p.outputs - 1) + (row & 32 ? p.outputs : 0);
            else
                o = min(w.n0 + row, p.outputs - 1);
            src[q] = wg + o * p.w_row;
        }
#pragma unroll
        for (int q = 0; q < C::QX; q++) {
            const int row = min(at.row(q), w.r.count - 1);
            const int from = EXT ? w.r.first + row : max(x_of(p, w.r.first + row, places[side][0][row]), 0);
            src[C::QW + q] = p.x + from * p.x_row + w.k_lo + at.piece;
        }
#pragma unroll
        for (int j = 0; j < C::FM; j++) {
            const int row = at.wm * (C::M / C::WM) + j * 32 + at.col, in = min(row, w.r.count - 1), e = w.r.first + in;
            to[j] = OUT == 0 || EXT ? e : y_of(p, e, places[side][1][in]);
            if (row >= w.r.count || (OUT != 0 && !EXT && x_of(p, e, places[side][0][in]) < 0)) to[j] = -1;
        }
    };
    if (t >= walk.end) return;
    Work w = work_of(t);
    ask(w, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    barrier();
    aim(w, 0);
    if (!EXT) begin<C>(at, src, w.steps);
    for (int side = 0;; side ^= 1) {
        // while the first stages are on their way: what the next tile is
        const Work now = w;
        t += walk.step;
        const bool again = t < walk.end;
        if (again) {
            w = work_of(t);
            ask(w, side ^ 1);
        }
        acc.clear();
        const int n0 = now.n0 + at.wn * (kOutN / C::WN);
        if constexpr (EXT) {
            // the adapters as more inputs: each one's b beside the rows' h, which is zero in rows of another
            constexpr int kIds = (C::M + 63) / 64, kParts = kHParts<T, OUT>;
            int ids[kIds], own[C::QX];  // of the tile's rows, a lane each; and of the rows that this lane loads
#pragma unroll
            for (int i = 0; i < kIds; i++) {
                const int row = i * 64 + at.lane;
                ids[i] = adapter_in(p, places[side][0][min(row, now.r.count - 1)]);
            }
#pragma unroll
            for (int q = 0; q < C::QX; q++) own[q] = adapter_in(p, places[side][0][min(at.row(q), now.r.count - 1)]);
            bool any = false;
            for (int id = next_adapter(ids, -1); id != INT32_MAX; id = next_adapter(ids, id)) {
                any = true;
                for (int k0 = 0; k0 < kParts * p.rank; k0 += K)
                    run_alone<T, C>(at, acc, [&](int q, uint16_t* to) {
                        const int k = k0 + at.piece;  // of a row of h2: each eight of b meet all their parts
                        if (q < C::QW) {
                            const int o = min(now.n0 + at.row(q), p.outputs - 1);
                            piece_or_zero(at, k < kParts * p.rank, p.b + ((int64_t)id * p.outputs + o) * p.rank + k / (8 * kParts) * 8, to);
                        } else {
                            const int row = now.r.first + min(at.row(q - C::QW), now.r.count - 1);
                            piece_or_zero(at, k < kParts * p.rank && own[q - C::QW] == id, p.h2 + (int64_t)row * (kParts * p.rank) + k, to);
                        }
                    });
            }
            if (any) {
                float size = 0.0f;
#pragma unroll
                for (int j = 0; j < C::FM; j++) {
                    const int row = min(at.wm * (C::M / C::WM) + j * 32 + at.col, now.r.count - 1);
                    const float unit = T == KK_F16 && adapter_in(p, places[side][0][row]) >= 0 ? p.h_unit[now.r.first + row] : 1.0f;
#pragma unroll
                    for (int n = 0; n < C::FN; n++)
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            size += acc.sum[n][j][k] * 0.0f;
                            if constexpr (T == KK_F16) acc.sum[n][j][k] *= unit;
                        }
                }
                // Zero times an infinity or NaN of one adapter's b is not zero in the rows of another, and an infinity of b times the parts of
                // an h, of which one is zero or of the other sign, is NaN.
                if (__ballot(size != 0.0f)) add_apart<T, C>(p, at, now.r, n0, places[side][0], acc);
            }
            barrier();
            begin<C>(at, src, now.steps);
        }
        int quad = at.half * 4;
        asm volatile("" : "+v"(quad));  // what depends on it is computed where it is used: kept over the loop it would go to scratch
        if (OUT != 0 && p.bias) {
            const float* bias = p.bias + (int64_t)now.r.g * p.outputs * (GATED ? 2 : 1);
#pragma unroll
            for (int i = 0; i < C::FN; i++)
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const int o = min(n0 + (GATED ? i / 2 : i) * 32 + k / 4 * 8 + quad + k % 4, p.outputs - 1);
                    const float b = bias[GATED && i % 2 ? p.outputs + o : o];
#pragma unroll
                    for (int j = 0; j < C::FM; j++) acc.sum[i][j][k] += b;
                }
        }
        if (now.rest)  // the inputs behind the last whole stage
            run_alone<T, C>(at, acc, [&](int q, uint16_t* to) {
                piece_or_zero(at, at.piece < now.rest, src[q] + (now.steps - min(C::S - 1, now.steps)) * K, to);
            });
        run_stages<T, C>(at, src, now.steps, at.wm * (C::M / C::WM) < now.r.count, acc);

        // the next tile's first stages are on their way while this one's results are stored
        int done[C::FM];
#pragma unroll
        for (int j = 0; j < C::FM; j++) done[j] = to[j];
        barrier();  // all waves have read the last stage, and the next tile's places are there
        if (again) {
            aim(w, side ^ 1);
            if (!EXT) begin<C>(at, src, w.steps);
        }
#pragma unroll
        for (int j = 0; j < C::FM; j++) {
#pragma unroll
            for (int i = 0; i < C::FN; i += GATED ? 2 : 1) {
                __builtin_amdgcn_sched_barrier(0);  // one piece at a time: the sums fill the registers
                const int o = n0 + i * (GATED ? 16 : 32);
                float v[4][4];
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        v[q][k] = acc.sum[i][j][4 * q + k];
                        if constexpr (GATED) v[q][k] = gated(p.gate, v[q][k], acc.sum[i + 1][j][4 * q + k]);
                    }
                if constexpr (OUT == 0) {
                    if (done[j] < 0) continue;
                    float* part = p.part + ((int64_t)now.split * p.entries + done[j]) * p.outputs;
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int at_o = o + q * 8 + quad, left = p.outputs - at_o;
                        if (left > 0) store4<KK_F32>(part, at_o, p.outputs % 4 == 0, left, v[q]);
                    }
                } else if (OUT != KK_F32 && p.y_vec == 2 && o + 32 <= p.outputs) {
                    // two quads of a row on two lanes 32 apart to eight outputs on each
#pragma unroll
                    for (int q = 0; q < 4; q += 2) {
                        uint32_t s[2][2];
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int k = 0; k < 2; k++)
                                s[h][k] = (uint32_t)ElemOf<T>::store(v[q + h][2 * k]) | (uint32_t)ElemOf<T>::store(v[q + h][2 * k + 1]) << 16;
                        const auto a = __builtin_amdgcn_permlane32_swap(s[0][0], s[1][0], false, false);
                        const auto b = __builtin_amdgcn_permlane32_swap(s[0][1], s[1][1], false, false);
                        if (done[j] >= 0) *(uint4*)((uint16_t*)p.y + done[j] * p.y_row + o + q * 8 + quad * 2) = uint4{a[0], b[0], a[1], b[1]};
                    }
                } else if (done[j] >= 0) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int at_o = o + q * 8 + quad, left = p.outputs - at_o;
                        if (left > 0) store4<OUT == 0 ? KK_F32 : OUT>(p.y, done[j] * p.y_row + at_o, p.y_vec, left, v[q]);
                    }
                }
            }
        }
        if (!again) break;
    }
}

// ------------------------------------------------------------------ adapters

// h of many rows, summed over its parts of the inputs, as parts of 16 bits: 32 lanes a row.  The products stay those of 16-bit operands; one
// part alone would lose up to 2^-8 of h.  6 us for 12,661 rows of 64.
template <int T, int PARTS>
__global__ void __launch_bounds__(256) halves_kernel(ProductDev p) {
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), sub = threadIdx.x & 31;
    if (row >= p.entries || adapter_of(p, row) < 0) return;  // 32 lanes together
    float v[KK_MOST_RANK / 32], top = 0.0f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < KK_MOST_RANK / 32; i++) {
        v[i] = 0.0f;
        if (sub + 32 * i < p.rank)
            for (int s = 0; s < p.h_splits; s++) v[i] += p.h[((int64_t)s * p.entries + row) * p.rank + sub + 32 * i];
        top = fmaxf(top, fabsf(v[i]));
        nan |= v[i] != v[i];
    }
    nan = (uint32_t)(__ballot(nan) >> (threadIdx.x & 32)) != 0;  // of the row
    float down = 1.0f, unit = 1.0f;
    if constexpr (T == KK_F16) {
        // f16 in units of 2^(e - 14), e the exponent of the row's largest: neither part leaves its range
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        const int e = min(max((int)(__float_as_uint(top) >> 23) & 255, 27), 254);
        down = __uint_as_float((uint32_t)(268 - e) << 23), unit = __uint_as_float((uint32_t)(e - 14) << 23);
    }
    if (sub == 0) p.h_unit[row] = nan ? NAN : unit;
#pragma unroll
    for (int i = 0; i < KK_MOST_RANK / 32; i++) {
        const int k = sub + 32 * i;
        if (k >= p.rank) continue;
        uint16_t* to = p.h2 + (int64_t)row * (PARTS * p.rank) + k / 8 * (8 * PARTS) + k % 8;
        float left = v[i] * down;
#pragma unroll
        for (int n = 0; n < PARTS; n++) {
            to[8 * n] = ElemOf<T>::store(left);
            left -= ElemOf<T>::load(to[8 * n]);
            if (!(fabsf(left) < INFINITY)) left = 0.0f;  // behind an infinity nothing is left, and not inf - inf
        }
    }
}

// y = the sum of the parts + bias + b h.  A block takes one row and 256 outputs, whose rows of b follow each other in memory: they are
// read in 16-byte pieces thread after thread, and the pieces' sums put together through LDS.  All its time is latency, so every load that
// waits for nothing is made first: 3.9 us for one row of 4,096 outputs, 8.4 for 96 rows of 6,144 (rank 32; 38 MB of b, 16 of them
// from memory).
template <int T, int OUT>
__global__ void __launch_bounds__(256) expand_kernel(ProductDev p) {
    constexpr int kAhead = 4;
    __shared__ __align__(16) float h[KK_MOST_RANK];
    extern __shared__ float sums[];  // [256][rank / 8, made odd]
    const int row = blockIdx.x / p.tiles_n, o0 = blockIdx.x % p.tiles_n * 256, tid = threadIdx.x;
    const int o = min(o0 + tid, p.outputs - 1);
    const int id = p.adapters ? adapter_of(p, row) : -1, pieces = p.rank / 8, ld = pieces | 1;
    float part[kAhead], own = p.bias ? p.bias[o] : 0.0f, hk = 0.0f;
    auto load_part = [&](int s) { return p.part[((int64_t)min(s, p.splits - 1) * p.entries + row) * p.outputs + o]; };
#pragma unroll
    for (int s = 0; s < kAhead; s++) part[s] = load_part(s);
    if (tid < p.rank)
        for (int s = 0; s < p.h_splits; s++) hk += p.h[((int64_t)s * p.entries + row) * p.rank + tid];
    for (int s = 0; s < p.splits; s += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (s) part[i] = load_part(s + i);
            if (s + i < p.splits) own += part[i];
        }
    }
    if (id >= 0) {
        const uint16_t* b = p.b + ((int64_t)id * p.outputs + o0) * p.rank;
        const int all = min(256, p.outputs - o0) * pieces;
        uint4 q[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) q[j] = *(const uint4*)(b + (int64_t)min(tid + j * 256, all - 1) * 8);
        if (tid < p.rank) h[tid] = hk;
        __syncthreads();
        for (int i0 = tid; i0 < all; i0 += 256 * kAhead) {
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const int i = i0 + j * 256;
                if (i >= all) break;
                if (i0 != tid) q[j] = *(const uint4*)(b + (int64_t)i * 8);
                uint16_t e[8];
                __builtin_memcpy(e, &q[j], 16);
                const int at = i / pieces, piece = i - at * pieces;
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++) v = fmaf(ElemOf<T>::load(e[k]), h[piece * 8 + k], v);
                sums[at * ld + piece] = v;
            }
        }
        __syncthreads();
        for (int k = 0; k < pieces; k++) own += sums[tid * ld + k];
    }
    if (o0 + tid < p.outputs) ((typename ElemOf<OUT>::type*)p.y)[(int64_t)row * p.y_row + o] = ElemOf<OUT>::store(own);
}

// ------------------------------------------------------------------ launches

typedef Tile<128, 64, 2, 2, 64, 3, 2> Tile64;
typedef Tile<64, 128, 2, 2, 64, 3, 2> Tile128;
typedef Tile<256, 128, 2, 4, 64, 3, 1> Tile128Wide;
typedef Tile<256, 256, 2, 4, 32, 4, 1> Tile256;

template <int T, class C, bool GATED, bool EXT, int OUT>
hipError_t run_tile(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    const size_t lds = d.start ? 2 * ((size_t)d.groups + 1) * 4 : 0;
    return launch(product_kernel<T, C, GATED, EXT, OUT>, dim3((unsigned)(d.blocks + (OUT == 0 ? p.shrink : 0))), dim3(C::kThreads), lds, s, d);
}

void set_grid(ProductDev& d, const ProductPlan& p) {
    d.splits = p.splits, d.k_split = p.k_split, d.tiles = p.tiles, d.tiles_n = p.tiles_n, d.blocks = p.blocks;
}

}  // namespace

template <int T, bool GATED>
static hipError_t expert_run(const ProductDev& d, const ProductPlan& p, hipStream_t s) {
    if (p.tile == k64) return run_tile<T, Tile64, GATED, false, T>(d, p, s);
    if (p.tile == k128Wide) return run_tile<T, Tile128Wide, GATED, false, T>(d, p, s);
    return run_tile<T, Tile256, GATED, false, T>(d, p, s);
}

hipError_t launch_expert_product(const kk_expert_product_args& a, const ProductPlan& p, hipStream_t s) {
    ProductDev d{};
    d.x = (const uint16_t*)a.x, d.w = (const uint16_t*)a.w, d.x_row = a.x_row, d.w_row = a.w_row, d.w_group = a.w_group;
    d.x_rows = a.x_rows, d.y_rows = a.y_rows, d.y_row = a.y_row, d.bias = a.bias, d.y = a.y;
    d.start = a.start, d.x_place = a.x_place, d.y_place = a.y_place, d.fault = a.fault, d.x_inv = 1.0 / std::max(a.x_div, 1);
    d.entries = a.entries, d.groups = a.groups, d.inputs = a.inputs, d.outputs = a.outputs, d.gate = a.gate;
    d.y_vec = (uintptr_t)a.y % 16 == 0 && a.y_row % 8 == 0 ? 2 : (uintptr_t)a.y % 8 == 0 && a.y_row % 4 == 0;
    set_grid(d, p);
    if (a.type == KK_BF16) return d.gate ? expert_run<KK_BF16, true>(d, p, s) : expert_run<KK_BF16, false>(d, p, s);
    return d.gate ? expert_run<KK_F16, true>(d, p, s) : expert_run<KK_F16, false>(d, p, s);
}

template <int T, bool EXT, int OUT>
static hipError_t adapter_main(ProductDev d, const ProductPlan& p, hipStream_t s) {
    set_grid(d, p);
    return p.tile == k64 ? run_tile<T, Tile64, false, EXT, OUT>(d, p, s) : run_tile<T, Tile128Wide, false, EXT, OUT>(d, p, s);
}

template <int T, int OUT>
static hipError_t adapter_run(ProductDev d, const AdapterPlan& r, hipStream_t s) {
    hipError_t rc;
    if (r.joined) {
        set_grid(d, r.main);
        rc = r.main.tile == k64 ? run_tile<T, Tile64, false, false, 0>(d, r.main, s) : run_tile<T, Tile128, false, false, 0>(d, r.main, s);
        if (rc != hipSuccess) return rc;
        d.tiles_n = (int)ceil_div(d.outputs, 256);
        return launch(expand_kernel<T, OUT>, dim3((unsigned)((int64_t)d.entries * d.tiles_n)), dim3(256), 256 * ((size_t)d.rank / 8 | 1) * 4, s, d);
    }
    if (d.adapters) {
        rc = launch(shrink_kernel<T, Tile128>, dim3((unsigned)r.main.shrink), dim3(Tile128::kThreads), 0, s, d);
        if (rc == hipSuccess) rc = launch(halves_kernel<T, kHParts<T, OUT>>, dim3((unsigned)ceil_div(d.entries, 8)), dim3(256), 0, s, d);
        if (rc != hipSuccess) return rc;
    }
    ProductDev rest = d;
    d.entries = r.rows;
    rc = d.adapters ? adapter_main<T, true, OUT>(d, r.main, s) : adapter_main<T, false, OUT>(d, r.main, s);
    if (rc != hipSuccess || r.rows == rest.entries) return rc;
    const int e = OUT == KK_F32 ? 4 : 2;
    rest.x += r.rows * d.x_row, rest.y = (char*)d.y + r.rows * d.y_row * e, rest.entries -= r.rows;
    if (d.adapters) rest.adapter += r.rows, rest.h += (int64_t)r.rows * d.rank, rest.h2 += (int64_t)r.rows * kHParts<T, OUT> * d.rank, rest.h_unit += r.rows;
    return d.adapters ? adapter_main<T, true, OUT>(rest, r.rest, s) : adapter_main<T, false, OUT>(rest, r.rest, s);
}

hipError_t launch_adapter_product(const kk_adapter_product_args& a, const AdapterPlan& r, hipStream_t s) {
    ProductDev d{};
    d.x = (const uint16_t*)a.x, d.w = (const uint16_t*)a.w, d.x_row = a.x_row, d.w_row = a.w_row;
    d.x_rows = d.y_rows = a.rows, d.y_row = a.y_row, d.bias = a.bias, d.y = a.y, d.fault = a.fault;
    d.entries = a.rows, d.groups = 1, d.inputs = a.inputs, d.outputs = a.outputs;
    const int e = a.out_type == KK_F32 ? 4 : 2;
    d.y_vec = e == 2 && (uintptr_t)a.y % 16 == 0 && a.y_row % 8 == 0 ? 2 : (uintptr_t)a.y % (4 * e) == 0 && a.y_row % 4 == 0;
    char* ws = (char*)a.workspace;
    d.adapters = a.adapters;
    if (a.adapters) {
        d.a = (const uint16_t*)a.a, d.b = (const uint16_t*)a.b, d.scale = a.scale, d.adapter = a.adapter, d.rank = a.rank;
        d.h = (float*)ws, d.h2 = (uint16_t*)(ws + r.ws_h2), d.h_unit = (float*)(ws + r.ws_unit);
        d.slots = r.slots, d.h_splits = r.h_splits, d.h_k = r.h_k, d.h_rows = a.rows;
    }
    d.part = (float*)(ws + r.ws_part);
    if (a.type == KK_BF16) return a.out_type == KK_F32 ? adapter_run<KK_BF16, KK_F32>(d, r, s) : adapter_run<KK_BF16, KK_BF16>(d, r, s);
    return a.out_type == KK_F32 ? adapter_run<KK_F16, KK_F32>(d, r, s) : adapter_run<KK_F16, KK_F16>(d, r, s);
}

}  // namespace kk
