// kk_kv.hip -- writing tokens into the 8-bit cache, and reading them back.
//
// Bound by memory: a value is read in 16 bits and written in 8 (and the other way round).  One block per (page of a
// sequence, head, K or V) holds the page's new tokens in registers, so their largest value, the page's scale and the
// stored bytes come from one pass; nothing of a page is shared between blocks.  V goes through LDS once more, because the
// cache holds a value's tokens next to each other: bytes are written [token][dim] and taken out as 4 x 4 byte blocks.
//
// Measured at 8 heads of 128 values, a kernel alone: writing 14,000 tokens of eight prompts (bf16, int8; 86 MB) 21 us, 4.1 TB/s,
// where the last-level cache holds their rows, 33 us, 2.6 TB/s, where it does not (a block reads 256 bytes of each packed row,
// whose neighbours other blocks read much later); reading them back 17 us, 5.1 TB/s; reading 32,001 tokens (197 MB) 31 us, 6.4 TB/s; one token each of 64 conversations 7.5 us, its
// 1,024 blocks' chain of length, page number, scale and bytes.  Writing was 29 us while each load waited for the one before and
// each value was checked for infinities: now all of a page's loads are in flight together, the sizes are compared on the bits, and
// only a block that holds an infinity or NaN checks its values.
#include "kk_kv.h"

namespace kk {
namespace {

// The page that a block works on.
template <int THREADS>
__device__ __forceinline__ bool kv_page(const KvCacheDev& c, const KvBatchDev& B, int per_seq, bool report, KvSeq& s, KvPage& p,
                                        int* found) {
    int i;
    if (per_seq) {
        const int b = blockIdx.x / per_seq;
        i = blockIdx.x - b * per_seq;
        if (!kv_seq(B, b, s)) {
            if (report && threadIdx.x == 0) kv_fault(c, KK_KV_BAD_BATCH);
            return false;
        }
    } else {
        i = kv_find<THREADS>(c, B, blockIdx.x, 1, kPage, 2, report && blockIdx.x == 0, s, found);
        if (i < 0) return false;
    }
    if (!kv_page_rows(s, i, p)) {
        if (report && threadIdx.x == 0 && s.m > s.len) kv_fault(c, KK_KV_BAD_BATCH);
        return false;
    }
    return true;
}

// Its number in the cache, or -1 for one that does not exist.
__device__ __forceinline__ int kv_page_id(const KvCacheDev& c, int id, bool report) {
    if (id >= 0 && id < c.pages) return id;
    if (report && threadIdx.x == 0) kv_fault(c, KK_KV_BAD_PAGE);
    return -1;
}

// 4 x 4 bytes transposed: o[i] byte j = w[j] byte i.
__device__ __forceinline__ void transpose4(const uint32_t w[4], uint32_t o[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    o[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    o[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    o[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    o[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

__device__ __forceinline__ uint32_t byte_mask(int first, int lo, int hi) {  // bytes first..first+3 that lie in [lo, hi)
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (first + i >= lo && first + i < hi) m |= 0xffu << (8 * i);
    return m;
}

constexpr int kKvThreads = 256;

template <class E>
__device__ __forceinline__ E bits_of(uint32_t u) {
    if constexpr (sizeof(E) == 4)
        return __uint_as_float(u);
    else
        return (E)u;
}

// The largest of a thread's values by their bits without signs, of those below `limit`.
template <int T, int N>
__device__ __forceinline__ uint32_t raw_max(const typename ElemOf<T>::type (*raw)[8], uint32_t limit) {
    if constexpr (T == KK_F32) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t u = __float_as_uint(raw[j][i]) & ElemOf<T>::mask;
                m = max(m, u < limit ? u : 0u);
            }
        return m;
    } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 m = {0, 0};
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                u16x2 u = {(uint16_t)(raw[j][i] & ElemOf<T>::mask), (uint16_t)(raw[j][i + 1] & ElemOf<T>::mask)};
                if (limit != ~0u) u = u16x2{u[0] < limit ? u[0] : (uint16_t)0, u[1] < limit ? u[1] : (uint16_t)0};
                m = __builtin_elementwise_max(m, u);
            }
        return max((uint32_t)m[0], (uint32_t)m[1]);
    }
}

// The largest over the block's threads; `words`: one of LDS a wave, not used by anything before.
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* words) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, k));
    if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = m;
    __syncthreads();
    m = words[0];
#pragma unroll
    for (int i = 1; i < kKvThreads / 64; i++) m = max(m, words[i]);
    return m;
}

template <int T, int CT, int D>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(KvCacheDev c, KvBatchDev B, KvRowsDev R, int per_seq) {
    constexpr int kChunks = D / 8, kMine = kPage * kChunks / kKvThreads;  // 8-value chunks of a token, of a thread
    constexpr int kLd = D + 4;                                           // bytes of a token's row in LDS
    __shared__ int found[2];
    __shared__ uint32_t block_top[2 * kKvThreads / 64];
    __shared__ uint32_t lds[kPage * kLd / 4];
    const int head = blockIdx.y >> 1, is_v = blockIdx.y & 1, tid = threadIdx.x;
    KvSeq s;
    KvPage p;
    if (!kv_page<kKvThreads>(c, B, per_seq, blockIdx.y == 0, s, p, found)) return;
    int id = B.table[s.b * B.stride + p.at];  // used behind the loads of the new tokens
    const void* src = is_v ? R.v : R.k;
    const int64_t row_step = is_v ? R.v_row : R.k_row, head_step = is_v ? R.v_head : R.k_head;
    const bool vec = is_v ? R.v_vec : R.k_vec;
    // every load before the first is used: threads whose slot is not written load the nearest one that is, and drop it
    typedef typename ElemOf<T>::type E;
    E raw[kMine][8];
    const E* from = (const E*)src + head * head_step;
#pragma unroll
    for (int j = 0; j < kMine; j++) {
        const int slot = (tid + j * kKvThreads) / kChunks, ch = (tid + j * kKvThreads) % kChunks;
        const E* q = from + (p.row0 + min(max(slot, p.lo), p.hi - 1) - p.lo) * row_step + ch * 8;
        if (vec) {
#pragma unroll
            for (int i = 0; i < 8; i += 16 / (int)sizeof(E)) {
                const uint4 w = *(const uint4*)(q + i);
                __builtin_memcpy(&raw[j][i], &w, 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) raw[j][i] = q[i];
        }
    }
    id = kv_page_id(c, id, blockIdx.y == 0);
    if (id < 0) return;
    float* scale_at = (is_v ? c.vs : c.ks) + (int64_t)id * c.heads + head;
    const float scale_was = p.lo ? *scale_at : 0.0f;
    uint8_t* page = (is_v ? c.v : c.k) + ((int64_t)id * c.heads + head) * (kPage * D);
    // The largest size, on the bits: two instructions for two values in 16 bits.  The other slots' threads hold values that are
    // written too and change nothing.  A block that holds infinities or NaN finds it again without them.
    const uint32_t most = block_max(raw_max<T, kMine>(raw, ~0u), block_top);
    const bool finite = most < ElemOf<T>::inf;
    const uint32_t top_bits = finite ? most : block_max(raw_max<T, kMine>(raw, ElemOf<T>::inf), block_top + kKvThreads / 64);
    const float top = sizeof(E) == 4 ? __uint_as_float(top_bits) : ElemOf<T>::load(bits_of<E>(top_bits));

    const float want = top > 0.0f ? fmaxf(top * (CT == KK_KV_E4M3 ? 1.0f / 448.0f : 1.0f / 127.0f), kScaleLeast) : 0.0f;
    const float scale = fmaxf(scale_was, want);
    const bool grown = p.lo > 0 && scale > scale_was;
    const float ratio = grown ? scale_was / scale : 1.0f;
    const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
    if (tid == 0) *scale_at = scale;
#pragma unroll
    for (int j = 0; j < kMine; j++) {
        const int slot = (tid + j * kKvThreads) / kChunks, ch = (tid + j * kKvThreads) % kChunks;
        f32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 4; i++) lo[i] = ElemOf<T>::load(raw[j][i]) * inv, hi[i] = ElemOf<T>::load(raw[j][4 + i]) * inv;
        const uint2 w = finite ? uint2{pack4_finite<CT>(lo), pack4_finite<CT>(hi)} : uint2{pack4<CT>(lo), pack4<CT>(hi)};
        if (is_v) {
            lds[slot * (kLd / 4) + ch * 2] = w.x;
            lds[slot * (kLd / 4) + ch * 2 + 1] = w.y;
            continue;
        }
        uint2* at = (uint2*)(page + slot * D + ch * 8);
        if (slot >= p.lo && slot < p.hi) {
            *at = w;
        } else if (grown && slot < p.lo) {
            uint2 o = *at;
            o.x = pack4<CT>(unpack4f<CT>(o.x) * ratio);
            o.y = pack4<CT>(unpack4f<CT>(o.y) * ratio);
            *at = o;
        }
    }
    if (!is_v) return;
    __syncthreads();
    // 16 tokens of 4 values a thread
    for (int t = tid; t < D; t += kKvThreads) {
        const int first = (t & 3) * 16, d = (t >> 2) * 4;
        if (first >= p.hi || (first + 16 <= p.lo && !grown)) continue;
        uint32_t o[4][4];
#pragma unroll
        for (int g = 0; g < 4; g++) {
            uint32_t w[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = lds[(first + 4 * g + i) * (kLd / 4) + d / 4];
            transpose4(w, y);
#pragma unroll
            for (int i = 0; i < 4; i++) o[i][g] = y[i];
        }
        const bool whole = first >= p.lo && first + 16 <= p.hi;
        if (!whole && !grown) {  // a few tokens: their bytes alone
            const int a = max(p.lo - first, 0), b = min(p.hi - first, 16);
#pragma unroll
            for (int k = 0; k < 16; k++)
                if (k >= a && k < b)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        page[(d + i) * kPage + first + k] = (uint8_t)(o[i][k >> 2] >> (8 * (k & 3)));
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint4* at = (uint4*)(page + (d + i) * kPage + first);
            uint32_t old[4] = {0, 0, 0, 0};
            if (!whole) __builtin_memcpy(old, at, 16);
            uint4 w;
            uint32_t* wp = (uint32_t*)&w;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t now = byte_mask(first + 4 * g, p.lo, p.hi), was = byte_mask(first + 4 * g, 0, p.lo);
                const uint32_t again = was ? pack4<CT>(unpack4f<CT>(old[g]) * ratio) : 0;
                wp[g] = (o[i][g] & now) | (again & was) | (old[g] & ~(now | was));
            }
            *at = w;
        }
    }
}

template <int T, int CT, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(KvCacheDev c, KvBatchDev B, KvRowsDev R, int per_seq) {
    constexpr int kChunks = D / 8, kMine = kPage * kChunks / kKvThreads;
    constexpr int kLd = D + 4;
    __shared__ int found[2];
    __shared__ uint32_t lds[kPage * kLd / 4];
    const int head = blockIdx.y >> 1, is_v = blockIdx.y & 1, tid = threadIdx.x;
    KvSeq s;
    KvPage p;
    if (!kv_page<kKvThreads>(c, B, per_seq, blockIdx.y == 0, s, p, found)) return;
    const int id = kv_page_id(c, B.table[s.b * B.stride + p.at], blockIdx.y == 0);
    const bool bad = id < 0;
    const int64_t at = (int64_t)(bad ? 0 : id) * c.heads + head;
    const float scale = bad ? __uint_as_float(0x7fc00000u) : (is_v ? c.vs : c.ks)[at];
    const uint8_t* page = (is_v ? c.v : c.k) + at * (kPage * D);
    void* dst = is_v ? R.v : R.k;
    const int64_t row_step = is_v ? R.v_row : R.k_row, head_step = is_v ? R.v_head : R.k_head;
    const bool vec = is_v ? R.v_vec : R.k_vec;
    if (is_v) {
        for (int t = tid; t < D; t += kKvThreads) {
            const int first = (t & 3) * 16, d = (t >> 2) * 4;
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; i++) __builtin_memcpy(w[i], page + (d + i) * kPage + first, 16);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t v[4] = {w[0][g], w[1][g], w[2][g], w[3][g]};
                uint32_t y[4];
                transpose4(v, y);
#pragma unroll
                for (int i = 0; i < 4; i++) lds[(first + 4 * g + i) * (kLd / 4) + d / 4] = y[i];
            }
        }
        __syncthreads();
    }
    uint2 w[kMine];
#pragma unroll
    for (int j = 0; j < kMine; j++) {
        const int slot = (tid + j * kKvThreads) / kChunks, ch = (tid + j * kKvThreads) % kChunks;
        w[j] = is_v ? uint2{lds[slot * (kLd / 4) + ch * 2], lds[slot * (kLd / 4) + ch * 2 + 1]}
                    : *(const uint2*)(page + slot * D + ch * 8);
    }
#pragma unroll
    for (int j = 0; j < kMine; j++) {
        const int slot = (tid + j * kKvThreads) / kChunks, ch = (tid + j * kKvThreads) % kChunks;
        if (slot < p.lo || slot >= p.hi) continue;
        const f32x4 a = unpack4f<CT>(w[j].x) * scale, b = unpack4f<CT>(w[j].y) * scale;
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        store_values<T, 8>(dst, (p.row0 + slot - p.lo) * row_step + head * head_step + ch * 8, vec, x);
    }
}

typedef void (*KvKernel)(KvCacheDev, KvBatchDev, KvRowsDev, int);

template <bool WRITE, int T, int CT>
KvKernel kv_kernel_of(int dim) {
#define KK_KV_CASE(D) \
    case D: return WRITE ? kv_write_kernel<T, CT, D> : kv_read_kernel<T, CT, D>;
    switch (dim) {
        KK_KV_CASE(64)
        KK_KV_CASE(96)
        KK_KV_CASE(128)
        KK_KV_CASE(192)
        KK_KV_CASE(256)
    }
#undef KK_KV_CASE
    return nullptr;
}
template <bool WRITE, int T>
KvKernel kv_kernel_of(int cache, int dim) {
    return cache == KK_KV_INT8 ? kv_kernel_of<WRITE, T, KK_KV_INT8>(dim) : kv_kernel_of<WRITE, T, KK_KV_E4M3>(dim);
}

template <bool WRITE>
hipError_t kv_launch(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_rows& r, hipStream_t s) {
    const int e = r.type == KK_F32 ? 4 : 2;
    auto whole = [&](const void* p, int64_t row, int64_t head) {
        return (uintptr_t)p % 16 == 0 && row * e % 16 == 0 && head * e % 16 == 0;
    };
    const KvRowsDev d{r.k, r.v, r.k_row, r.k_head, r.v_row, r.v_head, whole(r.k, r.k_row, r.k_head), whole(r.v, r.v_row, r.v_head)};
    const KvKernel k = r.type == KK_BF16  ? kv_kernel_of<WRITE, KK_BF16>(c.type, c.dim)
                       : r.type == KK_F16 ? kv_kernel_of<WRITE, KK_F16>(c.type, c.dim)
                                          : kv_kernel_of<WRITE, KK_F32>(c.type, c.dim);
    const KvTiles t = kv_tiles(b);
    return launch(k, dim3((unsigned)t.tiles, 2 * (unsigned)c.heads), dim3(kKvThreads), 0, s, kv_dev(c), kv_dev(b), d, t.per_seq);
}

}  // namespace

hipError_t launch_kv_write(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_rows& r, hipStream_t s) {
    return kv_launch<true>(c, b, r, s);
}
hipError_t launch_kv_read(const kk_kv_cache& c, const kk_kv_batch& b, const kk_kv_rows& r, hipStream_t s) {
    return kv_launch<false>(c, b, r, s);
}

}  // namespace kk
