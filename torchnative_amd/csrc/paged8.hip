// The paged 8-bit key/value cache: the writer and the reader of its rows
// (tnhip.h describes the planes).
//
// Sixteen tokens of a head, a block, share a scale, so that a row that joins a
// block may raise it and with it re-round the codes of the others. A wave owns
// a block's part of a call, the rows that enter it (they lie within sixteen rows
// of the call): it holds them in registers while it finds their largest size,
// then writes them and, where the scale grew, the block's other codes.
#include "paged.h"

#include <algorithm>
#include <cmath>

namespace tn {
namespace {

constexpr float MIN_SCALE = 1.1754943508222875e-38f;  // 2^-126

struct Row8Args {
    Pages8 c;
    const void *k, *v;
    void *ko, *vo;
    int64_t stride;
    const int32_t* slots;
    int64_t m;
    int window;  // append: rows whose blocks a wave takes
};

// The plane row (of D bytes) of a slot and head: in v_codes, of its block's first byte
// if the slot is the block's first.
__device__ inline int64_t plane_row(const Pages8& c, int slot, int h) {
    return (((int64_t)(slot >> c.shift) * c.H + h) << c.shift) + (slot & ((1 << c.shift) - 1));
}

__device__ inline int checked_slot(const Pages8& c, int slot) {
    return slot >= 0 && (slot >> c.shift) < c.pages ? slot : -1;
}

// Eight consecutive elements at any element.
template <int DT>
__device__ inline void load8(const void* p, int64_t i, float (&v)[8]) {
    float a[4], b[4];
    load4<DT>(p, i, a);
    load4<DT>(p, i + 4, b);
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = a[j], v[4 + j] = b[j];
}

// The byte of a value under 1 / scale: NaN as 0, infinities as the largest codes.
__device__ inline uint32_t byte_of(float v, float inv) {
    float c = v * inv;
    c = c == c ? fminf(fmaxf(rintf(c), -127.0f), 127.0f) : 0.0f;
    return (uint32_t)((int)c + 128);
}

// The bytes of a dword under a scale that grew by 1 / ratio.
__device__ inline uint32_t lowered(uint32_t w, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int c = (int)(w >> (8 * j) & 0xffu) - 128;
        r |= (uint32_t)((int)rintf((float)c * ratio) + 128) << (8 * j);
    }
    return r;
}

// A wave takes the blocks that rows of its window enter first, one after another, of one
// head, of K or of V: the rows of a block lie within sixteen rows of the call.
template <int DT, int NB>
__global__ __launch_bounds__(256) void k_append8(const Row8Args a) {
    constexpr int D = 32 * NB, C = D / 8;  // pieces of eight elements a row; NB of 64 lanes cover 16 rows
    __shared__ __align__(16) uint8_t tile[4][16 * D];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y;
    const bool v = blockIdx.z;
    const void* src = v ? a.v : a.k;
    uint8_t* plane = v ? a.c.vc : a.c.kc;
    float* scales = v ? a.c.vs : a.c.ks;
    const int64_t t0 = ((int64_t)blockIdx.x * 4 + w) * a.window - 15;  // lane 0's row; the window is lane 15's and on
    if (t0 + 15 >= a.m) return;  // (no barrier below)
    const int64_t t = t0 + lane;
    const int slot = t >= 0 && t < a.m ? checked_slot(a.c, a.slots[t]) : -1;
    const int block = slot < 0 ? -1 - lane : slot >> 4;  // (of no row: its own)
    bool joins = slot < 0, twice = false;
#pragma unroll
    for (int j = 1; j < 16; j++) {
        joins |= __shfl_up(block, j) == block && lane >= j;
        twice |= __shfl_down(slot, j) == slot && lane + j < 64;
    }
    uint64_t firsts = __ballot(!joins && lane >= 15 && lane < 15 + a.window);
    const uint64_t again = __ballot(twice && slot >= 0);
    while (firsts) {
        const int i = __ffsll((unsigned long long)firsts) - 1;  // the first row's lane
        firsts &= firsts - 1;
        const int b = __builtin_amdgcn_readlane(block, i);
        uint64_t rows = __ballot(block == b) & (0xffffull << i);  // lanes of its rows
        if (rows & again) {  // of a slot given twice the last counts
            bool drop = false;
#pragma unroll
            for (int j = 1; j < 16; j++)
                drop |= __shfl_down(slot, j) == slot && lane + j < 64 && (rows >> ((lane + j) & 63) & 1);
            rows &= ~__ballot(drop);
        }
        uint32_t tokens = 0;
        for (uint64_t left = rows; left; left &= left - 1)
            tokens |= 1u << (__builtin_amdgcn_readlane(slot, __ffsll((unsigned long long)left) - 1) & 15);
        float x[NB][8];
        float top = 0.0f;
        int token[NB];  // of this lane's piece of pass p, -1: none
#pragma unroll
        for (int p = 0; p < NB; p++) {
            const int it = p * 64 + lane, r = it / C, c = it % C;
            const int s = __shfl(slot, i + r);
            token[p] = rows >> (i + r) & 1 ? s & 15 : -1;
            if (token[p] >= 0) load8<DT>(src, (t0 + i + r) * a.stride + (int64_t)h * D + 8 * c, x[p]);
            else
#pragma unroll
                for (int j = 0; j < 8; j++) x[p][j] = 0.0f;
        }
#pragma unroll
        for (int p = 0; p < NB; p++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float s = fabsf(x[p][j]);
                top = s < INFINITY ? fmaxf(top, s) : top;
            }
        top = xor32_max(xor16_max(row16_max(top)));
        const int64_t prow = plane_row(a.c, b << 4, h);
        const bool fresh = tokens & 1;  // a row at its first slot begins a block anew
        float old = fresh ? 0.0f : scales[prow >> 4];
        if (!(old > 0.0f && old < INFINITY)) old = 0.0f;
        const float s = fmaxf(old, top > 0.0f ? fmaxf(top * (1.0f / 127.0f), MIN_SCALE) : 0.0f);
        const float inv = s > 0.0f ? 1.0f / s : 0.0f;
        const bool grew = !fresh && s > old;
        const float ratio = grew ? old / s : 1.0f;
        if (lane == 0) scales[prow >> 4] = s;
        uint8_t* to = plane + prow * D;
        uint8_t* mine = tile[w];
#pragma unroll
        for (int p = 0; p < NB; p++) {
            if (token[p] < 0) continue;
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++) o[j >> 2] |= byte_of(x[p][j], inv) << (8 * (j & 3));
            const int c = (p * 64 + lane) % C;
            *reinterpret_cast<uint2*>((v ? mine : to) + token[p] * D + 8 * c) = make_uint2(o[0], o[1]);
        }
        if (!v) {
            if (!grew) continue;
            for (int it = lane; it < 16 * C; it += 64) {
                if (tokens >> (it / C) & 1) continue;
                uint2* p = reinterpret_cast<uint2*>(to + 8 * it);
                const uint2 u = *p;
                *p = make_uint2(lowered(u.x, ratio), lowered(u.y, ratio));
            }
        } else {  // through LDS: sixteen tokens of an element leave together
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int d = lane; d < D; d += 64) {
                uint32_t o[4] = {0, 0, 0, 0};
                uint4* p = reinterpret_cast<uint4*>(to + d * 16);
                if (tokens != 0xffff) {
                    const uint4 u = *p;
                    o[0] = u.x, o[1] = u.y, o[2] = u.z, o[3] = u.w;
                    if (grew)
#pragma unroll
                        for (int j = 0; j < 4; j++) o[j] = lowered(o[j], ratio);
                }
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (tokens >> r & 1)
                        o[r >> 2] = (o[r >> 2] & ~(0xffu << (8 * (r & 3)))) | (uint32_t)mine[r * D + d] << (8 * (r & 3));
                *p = make_uint4(o[0], o[1], o[2], o[3]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// A workgroup takes 16 rows of one head, of K or of V: eight elements a thread.
template <int DT>
__global__ __launch_bounds__(256) void k_read8(const Row8Args a) {
    const int D = 32 * a.c.nb, C = D / 8, h = blockIdx.y;
    const bool v = blockIdx.z;
    const int64_t r0 = (int64_t)blockIdx.x * 16;
    for (int it = threadIdx.x; it < 16 * C; it += 256) {
        const int64_t t = r0 + it / C;
        const int c = it % C;
        if (t >= a.m) break;
        const int slot = checked_slot(a.c, a.slots[t]);
        float y[8];
        if (slot < 0) {
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = NAN;
        } else if (!v) {
            const int64_t row = plane_row(a.c, slot, h);
            const uint2 u = *reinterpret_cast<const uint2*>(a.c.kc + row * D + 8 * c);
            const float s = a.c.ks[row >> 4];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = (float)((int)((j < 4 ? u.x : u.y) >> (8 * (j & 3)) & 0xffu) - 128) * s;
        } else {
            const int64_t row = plane_row(a.c, slot & ~15, h);
            const uint8_t* p = a.c.vc + row * D + 8 * c * 16 + (slot & 15);
            const float s = a.c.vs[row >> 4];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = (float)((int)p[16 * j] - 128) * s;
        }
        void* out = v ? a.vo : a.ko;
        const int64_t o = (t * a.c.H + h) * D + 8 * c;
        const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
        store4<DT>(out, o, lo);
        store4<DT>(out, o + 4, hi);
    }
}

template <int DT>
void append_launch(hipStream_t st, const Row8Args& a) {
    const dim3 grid((unsigned)cdiv(a.m, 4 * a.window), (unsigned)a.c.H, 2);
#define TN_APPEND(NB)                                                                      \
    case NB:                                                                               \
        hipLaunchKernelGGL((k_append8<DT, NB>), grid, dim3(256), 0, st, a);                \
        break;
    switch (a.c.nb) {
        TN_APPEND(1) TN_APPEND(2) TN_APPEND(3) TN_APPEND(4) TN_APPEND(5) TN_APPEND(6) TN_APPEND(7) TN_APPEND(8)
    }
#undef TN_APPEND
}

template <int DT>
void read_launch(hipStream_t st, const Row8Args& a) {
    const dim3 grid((unsigned)cdiv(a.m, 16), (unsigned)a.c.H, 2);
    hipLaunchKernelGGL(k_read8<DT>, grid, dim3(256), 0, st, a);
}

tn_status row_check(const char* op, const tn_q8_cache* cache, int dtype, int64_t m, Row8Args* a) {
    TN_TRY(paged_check(op, cache, &a->c));
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, std::string(op) + ": rows must be float32, bfloat16 or float16");
    if (m < 0) return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    // up to 16 threads a row in a grid's first dimension, fewer than 2^32
    if (m > 1 << 27) return fail(TN_EVALUE, std::string(op) + ": shape too large");
    a->m = m;
    return TN_OK;
}

}  // namespace
}  // namespace tn

using namespace tn;

extern "C" {

tn_status tn_kv_append_q8(void* stream, const tn_q8_cache* cache, int dtype, const void* k, const void* v, int64_t m,
                          int64_t stride, const int32_t* slots) {
    const char* op = "kv_append_q8";
    Row8Args a{};
    TN_TRY(row_check(op, cache, dtype, m, &a));
    if (m > 1 && stride < (int64_t)a.c.H * a.c.nb * 32)
        return fail(TN_EINVAL, "kv_append_q8: the row stride is shorter than a row");
    if (m > 1 && stride > INT64_MAX / 8 / m) return fail(TN_EVALUE, "kv_append_q8: shape too large");
    if (m == 0) return TN_OK;
    if (!k || !v || !slots) return fail(TN_EVALUE, "kv_append_q8: null pointer");
    TN_TRY(paged_check_planes(op, a.c));
    a.k = k, a.v = v, a.stride = stride, a.slots = slots;
    a.window = m <= 1024 ? 1 : 16;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) append_launch<TN_F32>(st, a);
    else if (dtype == TN_BF16) append_launch<TN_BF16>(st, a);
    else append_launch<TN_F16>(st, a);
    TN_LAUNCHED();
    return TN_OK;
}

tn_status tn_kv_read_q8(void* stream, const tn_q8_cache* cache, const int32_t* slots, int64_t m, int dtype, void* k,
                        void* v) {
    const char* op = "kv_read_q8";
    Row8Args a{};
    TN_TRY(row_check(op, cache, dtype, m, &a));
    if (m == 0) return TN_OK;
    if (!k || !v || !slots) return fail(TN_EVALUE, "kv_read_q8: null pointer");
    TN_TRY(paged_check_planes(op, a.c));
    a.ko = k, a.vo = v, a.slots = slots;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) read_launch<TN_F32>(st, a);
    else if (dtype == TN_BF16) read_launch<TN_BF16>(st, a);
    else read_launch<TN_F16>(st, a);
    TN_LAUNCHED();
    return TN_OK;
}

}  // extern "C"
