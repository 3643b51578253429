// Pieces shared by the attention kernels over paged caches (paged_attn.hip,
// paged8_attn.hip): what a call of ragged rows is, f16 operands, loads.
#pragma once

#include "paged.h"

namespace tn {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// One call: what its kernels take. C: the cache's planes.
template <class C>
struct Ragged {
    C c;
    const void* q;
    void* out;
    float* lse;  // nullable
    const int32_t *row_start, *lens, *table;
    int64_t q_stride;
    int n, tokens, Hq, G, width, max_rows, max_len;  // G = Hq / H
    float sl2;        // scale * log2(e)
    int nsplit;       // splits of the keys in the kernel of few rows
    int few;          // requests of more folded rows are the kernel of many rows'; 0: all are
    float* part_o;    // [n][H][few][nsplit][D] and
    float2* part_ml;  // [n][H][few][nsplit], above one split
    float* many_o;    // many rows': [tokens][Hq][splits][D] and
    float2* many_ml;  // [tokens][Hq][splits], above one split
};

// Probabilities are kept at 2^P_BIAS times their size over the running maximum,
// which may lag by RESCALE_SLACK: at most 2^14, so that f16 holds them, and those
// far below the maximum stay out of its subnormal range as long as they count.
constexpr float P_BIAS = 6.0f;


// row_start[i], and request r's first row and number of rows: within the call's rows,
// whatever row_start holds.
template <class C>
TN_INLINE int start_of(const Ragged<C>& a, int i) { return min(max(a.row_start[i], 0), a.tokens); }
template <class C>
TN_INLINE int rows_of(const Ragged<C>& a, int r, int start) { return max(start_of(a, r + 1) - start, 0); }

// Pairs of f16 in a dword.
TN_INLINE h2 as_h2(uint32_t w) { return __builtin_bit_cast(h2, w); }
TN_INLINE uint32_t pk_mul(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, as_h2(a) * as_h2(b)); }
// a * b - c, rounded once: what c, the rounded product, lacks
TN_INLINE uint32_t pk_rest(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(as_h2(a), as_h2(b), -as_h2(c)));
}
TN_INLINE h8 as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h8, (u4){a, b, c, d});
}
TN_INLINE uint32_t pk_f16(float a, float b) { return El<true>::pack_p(a, b); }

// A pair of probabilities as f16 parts, and their sum, unrounded, onto l.
template <int PARTS>
TN_INLINE void split_p(float x, float y, uint32_t& hi, uint32_t& lo, float& l) {
    hi = pk_f16(x, y);
    if constexpr (PARTS == 2) {
        const h2 h = as_h2(hi);
        lo = pk_f16(x - (float)h[0], y - (float)h[1]);
    }
    l += x;
    l += y;
}

__device__ __attribute__((always_inline)) inline f32x4 mfma16(h8 a, h8 b, f32x4 c) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
    (void)a, (void)b;
    return c;
#endif
}

// A row's power of two: 2^-e with the largest element of size 2^e .. 2^(e+1), so
// that bf16 and f32 queries of any size fit f16, the smallest that count above its
// subnormals; 1 for rows of zeros, infinities and NaN.
__device__ inline float row_scale(float top) {
    const uint32_t e = (__builtin_bit_cast(uint32_t, top) >> 23) & 0xffu;
    // 2^(14 - (e - 127)), a normal number for e up to 254; a subnormal top counts as the smallest normal
    if (top == 0.0f || e == 255u) return 1.0f;
    const int x = 14 + 127 - (int)(e < 1u ? 1u : e) + 127;
    return __builtin_bit_cast(float, (uint32_t)(x > 254 ? 254 : x < 1 ? 1 : x) << 23);
}

template <int N>
__device__ __attribute__((always_inline)) inline void load_words(const void* p, uint32_t (&w)[N]) {
    // the widest pieces that N dwords come in; planes are 16-byte aligned, rows of N dwords N-aligned
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(4)));
    // (in the global address space, whatever the compiler can see of where p comes from)
#if __HIP_DEVICE_COMPILE__
#define TN_GLOBAL __attribute__((address_space(1)))
#else
#define TN_GLOBAL
#endif
    const TN_GLOBAL uint32_t* s = (const TN_GLOBAL uint32_t*)reinterpret_cast<uintptr_t>(p);
    constexpr int Q = N / 4 * 4;
#pragma unroll
    for (int i = 0; i < Q; i += 4) {
        const u4 x = *(const TN_GLOBAL u4*)(s + i);
#pragma unroll
        for (int j = 0; j < 4; j++) w[i + j] = x[j];
    }
    if constexpr (N % 4 >= 2) {
        const u2 x = *(const TN_GLOBAL u2*)(s + Q);
        w[Q] = x[0], w[Q + 1] = x[1];
    }
    if constexpr (N % 2) w[N - 1] = s[N - 1];
}

__device__ __attribute__((always_inline)) inline float half_of(uint32_t w, int i) {
    return (float)__builtin_bit_cast(h2, w)[i];
}

}  // namespace
}  // namespace tn
