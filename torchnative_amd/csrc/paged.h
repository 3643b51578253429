// The paged key/value caches of 4 bits (paged.hip, paged_attn.hip) and of 8
// (paged8.hip, paged8_attn.hip): their planes as the kernels index them, and the
// checks that every entry point makes.
#pragma once

#include "attn_common.h"

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

}  // namespace tn
