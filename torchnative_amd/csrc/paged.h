// The paged 4-bit key/value cache (paged.hip, paged_attn.hip): its planes as the
// kernels index them, and the checks that every entry point makes.
#pragma once

#include "tn_common.h"

namespace tn {

struct Pages {
    uint8_t* kc;   // [pages][H][S][4][nb][4]
    uint16_t* kd;  // [pages][H][S][nb]
    uint8_t* vc;   // [pages][H][S/8][16][nb][8]
    uint16_t* vd;  // [pages][H][S/8][nb][8]
    int pages, shift, H, nb;  // page size 1 << shift, head dim 32 nb
};

// The cache's own numbers, then (planes) its pointers.
tn_status paged_check(const char* op, const tn_q4_cache* cache, Pages* out);
tn_status paged_check_planes(const char* op, const Pages& c);

// The place of token i (0..7) among the eight bytes of v_codes: tokens 0 2 1 3 of
// each four, so that the halves of a dword masked to one nibble of each 16-bit
// half hold two consecutive tokens (bytes 0 and 2, bytes 1 and 3).
__host__ __device__ inline int v_place(int i) { return (i & 4) | ((i & 1) << 1) | ((i >> 1) & 1); }

}  // namespace tn
