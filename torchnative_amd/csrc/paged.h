// The paged key/value caches of 4 bits (paged.hip, paged_attn.hip) and of 8
// (paged8.hip, paged8_attn.hip): their planes as the kernels index them, and the
// checks that every entry point makes.
#pragma once

#include "attn_common.h"

#define TN_INLINE __device__ __attribute__((always_inline)) inline

namespace tn {

struct Pages {
    uint8_t* kc;   // [pages][H][S][4][nb][4]
    uint16_t* kd;  // [pages][H][S][nb]
    uint8_t* vc;   // [pages][H][S/8][16][nb][8]
    uint16_t* vd;  // [pages][H][S/8][nb][8]
    int pages, shift, H, nb;  // page size 1 << shift, head dim 32 nb
};

struct Pages8 {
    uint8_t* kc;  // [pages][H][S][D]
    float* ks;    // [pages][H][S/16]
    uint8_t* vc;  // [pages][H][S/16][D][16]
    float* vs;    // [pages][H][S/16]
    int pages, shift, H, nb;  // as above
};

// The cache's own numbers, then (planes) its pointers.
tn_status paged_check(const char* op, const tn_q4_cache* cache, Pages* out);
tn_status paged_check(const char* op, const tn_q8_cache* cache, Pages8* out);
tn_status paged_check_planes(const char* op, const Pages& c);
tn_status paged_check_planes(const char* op, const Pages8& c);

// The place of token i (0..7) among the eight bytes of v_codes: tokens 0 2 1 3 of
// each four, so that the halves of a dword masked to one nibble of each 16-bit
// half hold two consecutive tokens (bytes 0 and 2, bytes 1 and 3).
__host__ __device__ inline int v_place(int i) { return (i & 4) | ((i & 1) << 1) | ((i >> 1) & 1); }

// Four consecutive elements as floats, at any element.
template <int DT>
__device__ inline void load4(const void* p, int64_t i, float (&v)[4]) {
    if constexpr (DT == TN_F32) {
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
        const f4 x = *reinterpret_cast<const f4*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = x[j];
    } else {
        typedef uint16_t h4 __attribute__((ext_vector_type(4), aligned(2)));
        const h4 x = *reinterpret_cast<const h4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = DT == TN_BF16 ? bf16_to_f32(x[j]) : f16_bits_hw(x[j]);
    }
}

template <int DT>
__device__ inline void store4(void* p, int64_t i, const float (&v)[4]) {
    if constexpr (DT == TN_F32) {
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
        *reinterpret_cast<f4*>(static_cast<float*>(p) + i) = (f4){v[0], v[1], v[2], v[3]};
    } else {
        typedef uint32_t w2 __attribute__((ext_vector_type(2), aligned(2)));
        using E = El<DT == TN_F16>;
        *reinterpret_cast<w2*>(static_cast<uint16_t*>(p) + i) = (w2){E::pack_out(v[0], v[1]), E::pack_out(v[2], v[3])};
    }
}

// Eight consecutive elements of a row of type DT, at any element.
template <int DT>
struct Eight {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
    u4 w[DT == TN_F32 ? 2 : 1];
    TN_INLINE void load(const void* p, int64_t i) {
        const u4* s = reinterpret_cast<const u4*>(static_cast<const char*>(p) + i * (DT == TN_F32 ? 4 : 2));
        w[0] = s[0];
        if constexpr (DT == TN_F32) w[1] = s[1];
    }
    TN_INLINE void clear() { w[0] = w[DT == TN_F32 ? 1 : 0] = (u4){0, 0, 0, 0}; }
    TN_INLINE float get(int e) const {
        if constexpr (DT == TN_F32) return __uint_as_float(w[e >> 2][e & 3]);
        else return e & 1 ? El<DT == TN_F16>::hi(w[0][e >> 1]) : El<DT == TN_F16>::lo(w[0][e >> 1]);
    }
};

// Onto the largest size but NaN's, and onto what is NaN behind an infinity or a NaN.
template <int DT>
TN_INLINE void measure(const Eight<DT>& x, float& top, float& bad) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float v = x.get(j);
        top = fmaxf(top, fabsf(v));
        bad = fmaf(v, 0.0f, bad);
    }
}

// Four numbers of size 2^22 at most rounded to integers, halves to even, of which the low
// bytes: a sum with 1.5 * 2^23 has a step of one.
TN_INLINE uint32_t rounded_bytes(float a, float b, float c, float d) {
#if __HIP_DEVICE_COMPILE__
    constexpr float M = 12582912.0f;
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b + M), __float_as_uint(a + M), 0x0c0c0400u);
    return lo | __builtin_amdgcn_perm(__float_as_uint(d + M), __float_as_uint(c + M), 0x04000c0cu);
#else
    return (uint32_t)(a + b + c + d);
#endif
}

}  // namespace tn
