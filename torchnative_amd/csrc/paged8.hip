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
    int window;  // rows of a wave (append: rows whose blocks it takes)
};

// The plane row (of D bytes) of a slot and head: in v_codes, of its block's first byte
// if the slot is the block's first.
__device__ inline int64_t plane_row(const Pages8& c, int slot, int h) {
    return (((int64_t)(slot >> c.shift) * c.H + h) << c.shift) + (slot & ((1 << c.shift) - 1));
}

__device__ inline int checked_slot(const Pages8& c, int slot) {
    return slot >= 0 && (slot >> c.shift) < c.pages ? slot : -1;
}

// The bytes of four values under 1 / scale. ODD: values may be NaN, stored as 0 (infinities
// are held to the largest codes either way).
template <bool ODD>
TN_INLINE uint32_t bytes_of(const float (&v)[4], float inv) {
    float c[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        c[j] = v[j] * inv;
        if (ODD) c[j] = c[j] == c[j] ? c[j] : 0.0f;
        c[j] = fminf(fmaxf(c[j], -127.0f), 127.0f);
    }
    return rounded_bytes(c[0], c[1], c[2], c[3]) ^ 0x80808080u;
}

// Four bytes of each of a quad's lanes, transposed: byte i of lane j is byte j of lane i.
__device__ inline uint32_t quad_transposed(uint32_t w, int lane) {
#if __HIP_DEVICE_COMPILE__
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xf, 0xf, true);  // lane ^ 1
    const uint32_t v = __builtin_amdgcn_perm(y, w, lane & 1 ? 0x03070105u : 0x06020400u);
    const uint32_t z = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);  // lane ^ 2
    return __builtin_amdgcn_perm(z, v, lane & 2 ? 0x03020706u : 0x05040100u);
#else
    return w + (uint32_t)lane;
#endif
}

template <int DT>
__device__ inline void store8(void* p, int64_t i, const float (&lo)[4], const float (&hi)[4]) {
    if constexpr (DT == TN_F32) {
        store4<DT>(p, i, lo);
        store4<DT>(p, i + 4, hi);
    } else {
        typedef uint32_t w4 __attribute__((ext_vector_type(4), aligned(2)));
        using E = El<DT == TN_F16>;
        *reinterpret_cast<w4*>(static_cast<uint16_t*>(p) + i) =
            (w4){E::pack_out(lo[0], lo[1]), E::pack_out(lo[2], lo[3]), E::pack_out(hi[0], hi[1]), E::pack_out(hi[2], hi[3])};
    }
}

// A dword's bytes as codes.
__device__ inline void codes_of(uint32_t w, float scale, float (&y)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = (float)((int)(w >> (8 * j) & 0xffu) - 128) * scale;
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
// head, of K or of V: the rows of a block lie within sixteen rows of the call, so the fifteen
// ahead of the window tell which blocks are earlier waves' and the fifteen behind it what else
// enters. Bound by its bytes: 8192 bf16 rows of 8 heads of 128 elements, 50 MB, 10.2 to 11.4 us
// (4.4 to 4.9 TB/s, what a copy reaches); sixteen single rows 3.8 us, two trips to memory.
template <int DT, int NB>
__global__ __launch_bounds__(256) void k_append8(const Row8Args a) {
    // C pieces of eight elements a row: NB of 64 lanes cover 16 rows; U of 64 elements a row
    constexpr int D = 32 * NB, C = D / 8, U = (D + 63) / 64;
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
    for (uint64_t left = __ballot(slot >= 0 && lane >= 15 && lane < 15 + a.window); left;) {
        const int i = __ffsll((unsigned long long)left) - 1, first = __builtin_amdgcn_readlane(slot, i), b = first >> 4;
        const uint64_t same = __ballot(slot >> 4 == b);
        left &= ~same;
        if (same & (0x7fffull << (i - 15))) continue;  // an earlier row's
        uint64_t rows = same & (0xffffull << i);  // lanes of the block's rows
        uint32_t tokens = (uint32_t)(rows >> i) << (first & 15);
        if (rows & ~__ballot(slot - first == lane - i)) {  // out of order; of a slot given twice the last counts
            tokens = 0;
            for (uint64_t t = rows; t;) {
                const int last = 63 - __clzll((long long)t);
                const uint32_t bit = 1u << (__builtin_amdgcn_readlane(slot, last) & 15);
                t &= ~(1ull << last);
                if (tokens & bit) rows &= ~(1ull << last);
                tokens |= bit;
            }
        }
        // all that the block's part needs is asked for at once
        const int64_t prow = plane_row(a.c, b << 4, h);
        const bool fresh = tokens & 1;  // a row at its first slot begins a block anew
        float old = fresh ? 0.0f : scales[prow >> 4];
        uint8_t* to = plane + prow * D;
        uint4 held[U];
        if (v && tokens != 0xffff)
#pragma unroll
            for (int u = 0; u < U; u++) held[u] = *reinterpret_cast<const uint4*>(to + 16 * min(64 * u + lane, D - 1));
        Eight<DT> x[NB];
        int token[NB];  // of this lane's piece of pass p, -1: none
#pragma unroll
        for (int p = 0; p < NB; p++) {
            const int it = p * 64 + lane, r = it / C, c = it % C;
            const int s = __shfl(slot, i + r);
            token[p] = rows >> (i + r) & 1 ? s & 15 : -1;
            if (token[p] >= 0) x[p].load(src, (t0 + i + r) * a.stride + (int64_t)h * D + 8 * c);
            else x[p].clear();
        }
        float top = 0.0f, bad = 0.0f;  // bad: NaN if a value is not finite
#pragma unroll
        for (int p = 0; p < NB; p++) measure(x[p], top, bad);
        const bool odd = __any(bad != bad);
        if (odd) {
            top = 0.0f;
#pragma unroll
            for (int p = 0; p < NB; p++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float s = fabsf(x[p].get(j));
                    top = s < INFINITY ? fmaxf(top, s) : top;
                }
        }
        top = xor32_max(xor16_max(row16_max(top)));
        if (!(old > 0.0f && old < INFINITY)) old = 0.0f;
        const float s = fmaxf(old, top > 0.0f ? fmaxf(top * (1.0f / 127.0f), MIN_SCALE) : 0.0f);
        const float inv = s > 0.0f ? 1.0f / s : 0.0f;
        const bool grew = !fresh && s > old;
        const float ratio = grew ? old / s : 1.0f;
        if (lane == 0) scales[prow >> 4] = s;
        uint8_t* mine = tile[w];
#pragma unroll
        for (int p = 0; p < NB; p++) {
            if (token[p] < 0) continue;
            uint32_t o[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float y[4] = {x[p].get(4 * e), x[p].get(4 * e + 1), x[p].get(4 * e + 2), x[p].get(4 * e + 3)};
                o[e] = odd ? bytes_of<true>(y, inv) : bytes_of<false>(y, inv);
            }
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
#pragma unroll
            for (int u = 0; u < U; u++) {  // (D is a multiple of a half wave: a quad's lanes go together)
                const int d = 64 * u + lane;
                if (d >= D) break;
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[j] = quad_transposed(*reinterpret_cast<const uint32_t*>(mine + (4 * j + (d & 3)) * D + (d & ~3)), lane);
                if (tokens != 0xffff) {
                    const uint32_t was[4] = {held[u].x, held[u].y, held[u].z, held[u].w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        // a byte of ones for each new token
                        const uint32_t bits = tokens >> (4 * j) & 15u, mask = (bits * 0x00204081u & 0x01010101u) * 0xffu;
                        const uint32_t w = grew ? lowered(was[j], ratio) : was[j];
                        o[j] = (o[j] & mask) | (w & ~mask);
                    }
                }
                *reinterpret_cast<uint4*>(to + d * 16) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
}

// A wave takes the rows of its window, of one head, of K or of V: K's eight elements a lane;
// of V all the rows of one block together, whose elements come as sixteen tokens and are
// turned in quads of lanes. 8192 rows as above 10.9 to 12.1 us, a byte at a time 24.
template <int DT, int NB>
__global__ __launch_bounds__(256) void k_read8(const Row8Args a) {
    constexpr int D = 32 * NB, C = D / 8, U = (D + 63) / 64;
    __shared__ int row_at[4][16];  // of a block's token: the wave's row that is to have it
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y;
    const int64_t t0 = ((int64_t)blockIdx.x * 4 + w) * a.window;
    if (t0 >= a.m) return;  // (no barrier below)
    const bool is_row = lane < a.window && t0 + lane < a.m;
    const int slot = is_row ? checked_slot(a.c, a.slots[t0 + lane]) : -1;
    if (blockIdx.z == 0) {
        uint2 u[NB];
        float s[NB];
#pragma unroll
        for (int p = 0; p < NB; p++) {
            if (p * 64 >= a.window * C) break;
            const int it = p * 64 + lane, at = __shfl(slot, it / C);
            u[p] = make_uint2(0, 0), s[p] = NAN;
            if (at < 0) continue;  // (a cache may have no row at all)
            const int64_t row = plane_row(a.c, at, h);
            u[p] = *reinterpret_cast<const uint2*>(a.c.kc + row * D + 8 * (it % C));
            s[p] = a.c.ks[row >> 4];
        }
#pragma unroll
        for (int p = 0; p < NB; p++) {
            if (p * 64 >= a.window * C) break;
            const int it = p * 64 + lane, r = it / C;
            if (r >= a.window || t0 + r >= a.m) continue;
            const int64_t o = ((t0 + r) * a.c.H + h) * D + 8 * (it % C);
            float lo[4], hi[4];
            codes_of(u[p].x, s[p], lo);
            codes_of(u[p].y, s[p], hi);
            store8<DT>(a.ko, o, lo, hi);
        }
        return;
    }
    auto put = [&](int r, int d, uint32_t word, float scale) __attribute__((always_inline)) {
        float y[4];
        codes_of(word, scale, y);
        store4<DT>(a.vo, ((t0 + r) * a.c.H + h) * D + d, y);
    };
    for (uint64_t left = __ballot(is_row && slot < 0); left; left &= left - 1)
        for (int d = 4 * lane; d < D; d += 256) put(__ffsll((unsigned long long)left) - 1, d, 0, NAN);
    for (uint64_t left = __ballot(slot >= 0); left;) {
        const int b = __builtin_amdgcn_readlane(slot, __ffsll((unsigned long long)left) - 1) >> 4;
        const int64_t row = plane_row(a.c, b << 4, h);
        uint4 u[U];
#pragma unroll
        for (int x = 0; x < U; x++)
            u[x] = *reinterpret_cast<const uint4*>(a.c.vc + row * D + 16 * min(64 * x + lane, D - 1));
        const float s = a.c.vs[row >> 4];
        int* at = row_at[w];
        const bool mine = (left >> lane & 1) && slot >> 4 == b;
        if (lane < 16) at[lane] = -1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (mine) at[slot & 15] = lane;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        left &= ~__ballot(mine && at[slot & 15] == lane);  // (of a slot given twice one row a time)
        int to[4];
#pragma unroll
        for (int j = 0; j < 4; j++) to[j] = at[4 * j + (lane & 3)];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int x = 0; x < U; x++) {
            const int d = 64 * x + (lane & ~3);
            const uint32_t held[4] = {u[x].x, u[x].y, u[x].z, u[x].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t word = quad_transposed(held[j], lane);
                if (to[j] >= 0 && d < D) put(to[j], d, word, s);
            }
        }
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
    const dim3 grid((unsigned)cdiv(a.m, 4 * a.window), (unsigned)a.c.H, 2);
#define TN_READ(NB)                                                                        \
    case NB:                                                                               \
        hipLaunchKernelGGL((k_read8<DT, NB>), grid, dim3(256), 0, st, a);                  \
        break;
    switch (a.c.nb) {
        TN_READ(1) TN_READ(2) TN_READ(3) TN_READ(4) TN_READ(5) TN_READ(6) TN_READ(7) TN_READ(8)
    }
#undef TN_READ
}

// Rows of a wave's window: as few as make no more waves than the compute units hold at once
// (WINDOW_WAVES), so that blocks of single tokens do not wait for one another, and sixteen, a
// block of a prompt, where there are many. Append and read back, 8 heads of 128 elements, us,
// windows of 1 / of 16 / by this rule: 16 single tokens 6.4 / 27 / 6.4, 512 27 / 37 / 18, 2048 92 / 58 /
// 50; a prompt of 256 rows 7.1 / 7.6 / 7.2, 1024 15.3 / 8.3 / 7.6, 4096 41 / 15.3 / 15.3.
constexpr int64_t WINDOW_WAVES = 4096;
int window_of(const Pages8& c, int64_t m) {
    int w = 1;
    while (w < 16 && cdiv(m, w) * c.H * 2 > WINDOW_WAVES) w *= 2;
    return w;
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
    a.window = window_of(a.c, m);
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
    a.window = window_of(a.c, m);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) read_launch<TN_F32>(st, a);
    else if (dtype == TN_BF16) read_launch<TN_BF16>(st, a);
    else read_launch<TN_F16>(st, a);
    TN_LAUNCHED();
    return TN_OK;
}

}  // extern "C"
