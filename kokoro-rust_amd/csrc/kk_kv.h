// kk_kv.h -- the operators over an 8-bit cache: what their kernels share, and how the host sizes them.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kk_common.h"
#include "kk_kv_index.h"
#include "kokoro_hip.h"

namespace kk {

constexpr float kScaleLeast = 0x1p-90f;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// kk_kv_cache, kk_kv_batch and kk_kv_rows as the kernels take them.
struct KvCacheDev {
    uint8_t *k, *v;
    float *ks, *vs;
    int heads, pages;
    int32_t* fault;
};
struct KvRowsDev {
    void *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    int k_vec, v_vec;  // 16-byte accesses
};

inline KvCacheDev kv_dev(const kk_kv_cache& c) {
    return {(uint8_t*)c.k, (uint8_t*)c.v, c.k_scale, c.v_scale, c.heads, c.pages, c.fault};
}
// ------------------------------------------------------------------ batches on the device

__device__ __forceinline__ void kv_fault(const KvCacheDev& c, int bit) {
    if (c.fault) atomicOr(c.fault, bit);
}

// Which sequence's tile a block works on (kv_tile_base).  Every thread of the block calls this; `found` is two words of LDS.
// Returns the tile's number in its sequence, or -1 (a number that no sequence uses, or a bad sequence).  Where row_start falls, two
// sequences may claim a tile: what is left in `found` is then checked against the sequence as any tile is.
template <int THREADS>
__device__ __forceinline__ int kv_find(const KvCacheDev& c, const KvBatchDev& B, int64_t tile, int64_t G, int M, int E,
                                       bool report, KvSeq& s, int* found) {
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < B.n; b += THREADS) {
        KvSeq t;
        const bool ok = kv_seq(B, b, t);
        if (!ok && report) kv_fault(c, KK_KV_BAD_BATCH);
        int i;
        if (ok && kv_tile_in(t, tile, G, M, E, i)) found[0] = b, found[1] = i;
    }
    __syncthreads();
    const int b = __builtin_amdgcn_readfirstlane(found[0]);  // scalar from here on
    if (b < 0) return -1;
    kv_seq(B, b, s);
    return __builtin_amdgcn_readfirstlane(found[1]);
}

// ------------------------------------------------------------------ stored numbers

// Two bytes each of two words to four f16 (exact for both types): e4m3 by the conversion, int8 through 1024 + (x + 128),
// whose f16 has the byte as its low mantissa bits.
template <int CT>
__device__ __forceinline__ void unpack4(uint32_t x, f16x2& lo, f16x2& hi) {
    if constexpr (CT == KK_KV_E4M3) {
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true));
    } else {
        const uint32_t y = x ^ 0x80808080u;
        const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u)) - off;
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u)) - off;
    }
}
// Eight bytes to an MFMA operand.
template <int CT>
__device__ __forceinline__ f16x8 unpack8(uint32_t a, uint32_t b) {
    f16x2 p, q, r, s;
    unpack4<CT>(a, p, q);
    unpack4<CT>(b, r, s);
    return f16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}
// Four bytes to f32.
template <int CT>
__device__ __forceinline__ f32x4 unpack4f(uint32_t x) {
    f16x2 lo, hi;
    unpack4<CT>(x, lo, hi);
    return f32x4{(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]};
}
// Four numbers in units of their scale to bytes: nearest even, clamped, NaN to 0.
template <int CT>
__device__ __forceinline__ uint32_t pack4(f32x4 x) {
    constexpr float top = CT == KK_KV_E4M3 ? 448.0f : 127.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -top), top) : 0.0f;
    if constexpr (CT == KK_KV_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) w |= ((uint32_t)(int)rintf(x[i]) & 0xffu) << (8 * i);
        return w;
    }
}

// The same for numbers that are finite and at most the largest stored one (and a rounding): int8 by adding 1.5 x 2^23, whose sum
// has the nearest even integer in its low bits.
template <int CT>
__device__ __forceinline__ uint32_t pack4_finite(f32x4 x) {
    if constexpr (CT == KK_KV_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma clang fp contract(off)
            const float r = x[i] + 12582912.0f;
            u[i] = __float_as_uint(r);
        }
        const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u);
        return __builtin_amdgcn_perm(b, a, 0x05040100u);
    }
}

// ------------------------------------------------------------------ values in 16 and 32 bits

// `mask`: of a value's bits without its sign, whose order is that of the sizes; from `inf` on they are no numbers.
template <int T>
struct ElemOf;
template <>
struct ElemOf<KK_BF16> {
    typedef uint16_t type;
    static constexpr uint32_t mask = 0x7fff, inf = 0x7f80;
    static __device__ __forceinline__ float load(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t store(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
};
template <>
struct ElemOf<KK_F16> {
    typedef uint16_t type;
    static constexpr uint32_t mask = 0x7fff, inf = 0x7c00;
    static __device__ __forceinline__ float load(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ uint16_t store(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};
template <>
struct ElemOf<KK_F32> {
    typedef float type;
    static constexpr uint32_t mask = 0x7fffffff, inf = 0x7f800000;
    static __device__ __forceinline__ float load(float v) { return v; }
    static __device__ __forceinline__ float store(float f) { return f; }
};

// A load of data that is read once: it does not displace what the caches hold for others.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint4 stream_load(const uint4* p) {
    const u32x4 v = __builtin_nontemporal_load((const u32x4*)p);
    return uint4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ uint2 stream_load(const uint2* p) {
    const u32x2 v = __builtin_nontemporal_load((const u32x2*)p);
    return uint2{v[0], v[1]};
}

// N values next to each other, as 16-byte accesses where `vec` says that they lie on such a boundary.
template <int T, int N>
__device__ __forceinline__ void store_values(void* base, int64_t at, bool vec, const float* x) {
    typedef typename ElemOf<T>::type E;
    constexpr int W = 16 / (int)sizeof(E);
    E* p = (E*)base + at;
    E e[N];
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = ElemOf<T>::store(x[i]);
    if (vec && N % W == 0) {
#pragma unroll
        for (int i = 0; i < N; i += W) {
            uint4 q;
            __builtin_memcpy(&q, e + i, 16);
            *(uint4*)(p + i) = q;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = e[i];
    }
}

// ------------------------------------------------------------------ host side

hipError_t launch_norm_rope(const kk_norm_rope& a, int n_cu, hipStream_t s);
hipError_t launch_kv_write(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_rows& r, hipStream_t s);
hipError_t launch_kv_read(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_rows& r, hipStream_t s);
hipError_t launch_kv_attention(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_attention_args& a,
                               const AttnPlan& p, hipStream_t s);

// What the operators use of a context (kk_engine.hip).
int ctx_device(const kk_ctx* ctx);
int ctx_cus(const kk_ctx* ctx);

// One launch, with its own status (hipGetLastError would also report an earlier call's error).
template <class... P, class... A>
inline hipError_t launch(void (*k)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s, A... a) {
    static_assert(sizeof...(P) == sizeof...(A), "a launch passes every parameter of its kernel");
    return [&](P... p) {
        void* args[] = {(void*)&p...};
        return hipLaunchKernel((const void*)k, grid, block, args, lds, s);
    }(a...);
}

}  // namespace kk
