// Rows in 8-bit integers under one scale a row, and the linear over them
// (tnhip.h: tn_i8_*).
//
// Both operands are int8 over the whole of K, so the product is one exact
// integer sum an output, on the int8 matrix core, and its only roundings are the
// epilogue's: y = ((float)sum * w_scale) * a_scale (+ bias). A row's bits thus
// do not depend on the tile, the split or the rows around it.
#include <algorithm>
#include <cmath>

#include "attn_common.h"  // LdsDma, wait_vmcnt, El
#include "paged.h"        // load4

namespace tn {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t MAX_K = 131072;         // 127 * 127 * k < 2^31
constexpr int64_t MAX_ROWS = (1 << 24) - 1;
constexpr float MIN_SCALE = 1.1754943508222875e-38f;  // 2^-126

__host__ __device__ inline int64_t pitch_of(int64_t k) { return (k + 63) / 64 * 64; }

// Rows of codes with their scales: [rows][pitch], [rows].
struct Codes {
    const int8_t* c;
    const float* s;
};

// The scale of a row whose largest finite size is `top`.
__device__ inline float scale_of(float top) { return top > 0.0f ? fmaxf(top * (1.0f / 127.0f), MIN_SCALE) : 0.0f; }

// Eight elements from i on of a row of k, zeros behind it.
template <int DT>
TN_INLINE void load_row8(const void* x, int64_t row, int i, int k, Eight<DT>& v) {
    if (i + 8 <= k) return v.load(x, row + i);
    v.clear();
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (i + j >= k) continue;
        if constexpr (DT == TN_F32) v.w[j >> 2][j & 3] = static_cast<const uint32_t*>(x)[row + i + j];
        else v.w[0][j >> 1] |= (uint32_t) static_cast<const uint16_t*>(x)[row + i + j] << (16 * (j & 1));
    }
}

// The eight codes of v under 1 / scale (0 for a row that is not finite). No value's is past
// +-127: the scale's two roundings and its inverse's leave 127 (1 + 2^-22) at most.
template <int DT>
TN_INLINE uint2 codes8(const Eight<DT>& v, float inv, bool odd) {
    if (odd) return make_uint2(0, 0);
    return make_uint2(rounded_bytes(v.get(0) * inv, v.get(1) * inv, v.get(2) * inv, v.get(3) * inv),
                      rounded_bytes(v.get(4) * inv, v.get(5) * inv, v.get(6) * inv, v.get(7) * inv));
}

// T threads a row, which hold up to eight times HOLD elements each and read what is past
// these again: a wave where it holds the row, so that nothing waits at a barrier. Bound by
// memory where rows are many (bf16, 4096 of 4096 elements 9.5 us, 5.3 TB/s; of 14336 36 us, 4.9),
// by a launch where few (sixteen of 4096 3.2 us).
template <int DT, int T, int HOLD>
__global__ __launch_bounds__(256) void k_i8_rows(const void* __restrict__ x, int m, int k, int8_t* __restrict__ codes,
                                                 float* __restrict__ scales) {
    constexpr int RW = 256 / T;
    __shared__ float red[4];
    __shared__ int bads[4];
    const int tid = threadIdx.x % T, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * RW + threadIdx.x / T;
    const bool on = row < m;
    const int64_t at = (on ? row : 0) * k;
    const int pitch = (int)pitch_of(k);
    Eight<DT> v[HOLD];
    float top = 0.0f, bad = 0.0f;
#pragma unroll
    for (int h = 0; h < HOLD; h++) load_row8<DT>(x, at, 8 * (h * T + tid), k, v[h]);
#pragma unroll
    for (int h = 0; h < HOLD; h++) measure(v[h], top, bad);
    for (int i = 8 * (HOLD * T + tid); i < k; i += 8 * T) {
        Eight<DT> u;
        load_row8<DT>(x, at, i, k, u);
        measure(u, top, bad);
    }
    top = xor32_max(xor16_max(row16_max(top)));
    bool odd = __any(bad != bad);
    if constexpr (T > 64) {
        if (lane == 0) red[w] = top, bads[w] = odd;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        odd = bads[0] | bads[1] | bads[2] | bads[3];
    }
    if (!on) return;
    const float s = scale_of(top), inv = s > 0.0f ? 1.0f / s : 0.0f;
    if (tid == 0) scales[row] = odd ? NAN : s;
    int8_t* out = codes + row * pitch;
#pragma unroll
    for (int h = 0; h < HOLD; h++) {
        const int i = 8 * (h * T + tid);
        if (i < pitch) *reinterpret_cast<uint2*>(out + i) = codes8(v[h], inv, odd);
    }
    for (int i = 8 * (HOLD * T + tid); i < pitch; i += 8 * T) {
        Eight<DT> u;
        load_row8<DT>(x, at, i, k, u);
        *reinterpret_cast<uint2*>(out + i) = codes8(u, inv, odd);
    }
}

struct MmArgs {
    Codes a, w;
    const float* bias;  // nullable
    void* y;
    int m, n, pitch, y_dtype;
};

typedef int i32x16 __attribute__((ext_vector_type(16)));

__device__ __attribute__((always_inline)) inline i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
#else
    (void)a, (void)b;
    return c;
#endif
}
__device__ __attribute__((always_inline)) inline i32x16 mfma_i8(i32x4 a, i32x4 b, i32x16 c) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
#else
    (void)a, (void)b;
    return c;
#endif
}

// The epilogue of one sum.
__device__ inline float finish(int sum, float sw, float sx, bool biased, float bias) {
    const float v = ((float)sum * sw) * sx;
    return biased ? v + bias : v;
}

// A lane of the lower half gives b and takes the upper half's a, which gives a and takes
// b: x, y are then the lower lanes' a of both halves (lower half) and the b of both (upper).
template <class V>
__device__ __attribute__((always_inline)) inline void trade(V a, V b, V& x, V& y) {
    const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false,
                                                    false);
    x = __builtin_bit_cast(V, (uint32_t)p[0]);
    y = __builtin_bit_cast(V, (uint32_t)p[1]);
}

// Up to eight consecutive elements, at any element.
__device__ __attribute__((always_inline)) inline void put8(float* to, const float (&y)[8], int count) {
    typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
    if (count >= 8) {
        *reinterpret_cast<v4*>(to) = (v4){y[0], y[1], y[2], y[3]};
        *reinterpret_cast<v4*>(to + 4) = (v4){y[4], y[5], y[6], y[7]};
        return;
    }
#pragma unroll
    for (int u = 0; u < 7; u++)
        if (u < count) to[u] = y[u];
}
__device__ __attribute__((always_inline)) inline void put8(uint16_t* to, const uint32_t (&y)[4], int count) {
    typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
    if (count >= 8) {
        *reinterpret_cast<v4*>(to) = (v4){y[0], y[1], y[2], y[3]};
        return;
    }
#pragma unroll
    for (int u = 0; u < 7; u++)
        if (u < count) to[u] = (uint16_t)(y[u / 2] >> (16 * (u & 1)));
}

// ---- many rows -----------------------------------------------------------------------
//
// A workgroup of WN x WM waves, each RT x CT tiles of 32 channels by 32 tokens (the
// weights are the product's rows, so that a lane's sums are runs of four channels of a
// token). K goes KB bytes a stage through a ring of NS stages in LDS, filled by loads
// that go straight there (KG groups of waves: a stage each has its own KB bytes, and the
// groups' sums are added up at the end); a row's 16-byte chunks lie permuted by its number, so that
// sixteen rows' chunks cover every bank. A step of 32 bytes of K is read while the step
// before it is multiplied; one barrier a stage.
template <int WN, int WM, int RT, int CT, int KB, int NS, int KG = 1>
struct Tile {
    static constexpr int W = WN * WM, BN = 32 * RT * WN, BM = 32 * CT * WM;  // waves of a group
    static constexpr int LW = BN * KB / 1024 / W, LX = BM * KB / 1024 / W;  // loads of a wave, a stage
    static_assert(LW * W * 1024 == BN * KB && LX * W * 1024 == BM * KB, "whole loads");
    static constexpr int PER = LW + LX, OX = BN * KB, PART = (BN + BM) * KB, STAGE = KG * PART, STEPS = KB / 32;
    static_assert(KG == 1 || NS * STAGE >= (KG - 1) * W * RT * CT * 4096, "room for the groups' sums");
    static constexpr int SIDE = BN > BM ? BN : BM;
    static_assert((NS - 2) * PER < 64, "loads in flight");
};

// The tile of tokens from m0 on and channels from n0 on. ring: NS * STAGE bytes; side: the
// weights' scales, the bias, the tokens' scales, of SIDE floats each.
template <int WN, int WM, int RT, int CT, int KB, int NS, int KG = 1>
__device__ __attribute__((always_inline)) inline void gemm_tile(const MmArgs& a, uint8_t* ring, float* side, int m0,
                                                                int n0) {
    using T = Tile<WN, WM, RT, CT, KB, NS, KG>;
    constexpr int W = T::W, CH = KB / 16, RPL = 1024 / KB;  // chunks of a row, rows of a load
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) % W, group = __builtin_amdgcn_readfirstlane(tid >> 6) / W;
    float *const side_w = side, *const side_b = side + T::SIDE, *const side_x = side + 2 * T::SIDE;
    const int pitch = a.pitch;
    const LdsDma rw(a.w.c + (int64_t)n0 * pitch, (uint32_t)(min(T::BN, a.n - n0) * pitch));
    const LdsDma rx(a.a.c + (int64_t)m0 * pitch, (uint32_t)(min(T::BM, a.m - m0) * pitch));
    // chunk c of row r lies at place c ^ swz(r)
    auto swz = [](int r) { return KB == 128 ? (r >> 1) & 7 : (r >> 2) & 3; };
    uint32_t vw[T::LW], vx[T::LX];
    int last[T::LW > T::LX ? T::LW : T::LX];  // this lane's chunk's first byte within a stage
#pragma unroll
    for (int j = 0; j < (T::LW > T::LX ? T::LW : T::LX); j++) {
        const int r = (j * W + wave) * RPL + lane / CH, c = (lane % CH) ^ swz(r);
        if (j < T::LW) vw[j] = (uint32_t)(r * pitch + c * 16);
        if (j < T::LX) vx[j] = (uint32_t)(r * pitch + c * 16);
        last[j] = c * 16;
    }
    auto issue = [&](int st, int slot) __attribute__((always_inline)) {
        uint8_t* const s = ring + slot * T::STAGE + group * T::PART;
        const int k = (st * KG + group) * KB;
        const bool cut = k + KB > pitch;  // rows end within the last stage
#pragma unroll
        for (int j = 0; j < T::LW; j++)
            rw.load16(cut && k + last[j] >= pitch ? BUF_OOB : vw[j] + (uint32_t)k, s + (j * W + wave) * 1024);
#pragma unroll
        for (int j = 0; j < T::LX; j++)
            rx.load16(cut && k + last[j] >= pitch ? BUF_OOB : vx[j] + (uint32_t)k, s + T::OX + (j * W + wave) * 1024);
    };
    const int r32 = lane & 31, hh = lane >> 5, wn = wave / WM * 32 * RT, wm = wave % WM * 32 * CT;
    const uint32_t base = (uint32_t)(hh ^ swz(r32)) * 16;
    uint32_t pw = (uint32_t)((wn + r32) * KB), px = (uint32_t)(T::OX + (wm + r32) * KB);
    struct Step {
        i32x4 w[RT], x[CT];
    } f[2];
    auto read = [&](const uint8_t* s, int step, Step& y) __attribute__((always_inline)) {
        const uint32_t o = base ^ (uint32_t)(32 * step);
#pragma unroll
        for (int i = 0; i < RT; i++) y.w[i] = *reinterpret_cast<const i32x4*>(s + pw + o + i * 32 * KB);
#pragma unroll
        for (int j = 0; j < CT; j++) y.x[j] = *reinterpret_cast<const i32x4*>(s + px + o + j * 32 * KB);
    };
    i32x16 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < CT; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
    auto multiply = [&](const Step& y) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j < CT; j++) acc[i][j] = mfma_i8(y.w[i], y.x[j], acc[i][j]);
    };
    const int nst = (pitch + KG * KB - 1) / (KG * KB);
    // stage st has landed for every wave, and every wave has read the stages before it
    auto landed = [&](int st) __attribute__((always_inline)) {
        if (st + NS - 2 < nst) wait_vmcnt<(NS - 2) * T::PER>();
        else wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    for (int st = 0; st < min(NS, nst); st++) issue(st, st);
    for (int i = tid; i < T::BN; i += 64 * W * KG) {
        side_w[i] = n0 + i < a.n ? a.w.s[n0 + i] : 0.0f;
        side_b[i] = a.bias && n0 + i < a.n ? a.bias[n0 + i] : 0.0f;
    }
    for (int i = tid; i < T::BM; i += 64 * W * KG) side_x[i] = m0 + i < a.m ? a.a.s[m0 + i] : 0.0f;
    // (the last of these stages is one more than the loop has in flight)
    if (nst >= NS) wait_vmcnt<(NS - 1) * T::PER>();
    else wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(ring + group * T::PART, 0, f[0]);
    int slot = 0;
    static_assert(T::STEPS % 2 == 0, "two sets of operands in turn");
    auto stage = [&](int st, bool more) __attribute__((always_inline)) {
        const uint8_t* const s = ring + slot * T::STAGE + group * T::PART;
        const int next = slot + 1 < NS ? slot + 1 : 0;
#pragma unroll
        for (int k = 0; k < T::STEPS; k++) {
            __builtin_amdgcn_sched_barrier(0);
            if (k + 1 < T::STEPS) read(s, k + 1, f[(k + 1) & 1]);
            else if (more) {
                landed(st + 1);
                if (st + NS < nst) issue(st + NS, slot);
                read(ring + next * T::STAGE + group * T::PART, 0, f[(k + 1) & 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
            multiply(f[k & 1]);
        }
        slot = next;
    };
    for (int st = 0; st + 1 < nst; st++) stage(st, true);
    stage(nst - 1, false);
    // the last products' wait states, whatever their first reader is
    __builtin_amdgcn_sched_barrier(0);
#if __HIP_DEVICE_COMPILE__
    asm volatile("s_nop 15\n\ts_nop 1");
#endif
    __builtin_amdgcn_sched_barrier(0);

    if constexpr (KG > 1) {  // the groups' sums, added up by the first
        i32x4* const sums = reinterpret_cast<i32x4*>(ring);
        __syncthreads();
        if (group) {
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int j = 0; j < CT; j++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        sums[((((group - 1) * W + wave) * RT + i) * CT + j) * 256 + e * 16 + lane] =
                            (i32x4){acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        }
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int o = 0; o < KG - 1; o++)
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int j = 0; j < CT; j++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const i32x4 v = sums[(((o * W + wave) * RT + i) * CT + j) * 256 + e * 16 + lane];
#pragma unroll
                        for (int u = 0; u < 4; u++) acc[i][j][e + u] += v[u];
                    }
    }

    // A lane's sums of a tile are channels 8 u + 4 hh .. + 3 (u = 0 .. 3) of its token: its
    // half trades with the other, so that it has eight in a row, twice.
    const bool whole = n0 + T::BN <= a.n;  // uniform
    auto leave = [&](auto type) __attribute__((always_inline)) {
        constexpr int DT = decltype(type)::value;
#pragma unroll
        for (int j = 0; j < CT; j++) {
            const int m = m0 + wm + 32 * j + r32;
            const float sx = side_x[wm + 32 * j + r32];
            const int64_t row = (int64_t)m * a.n;
#pragma unroll
            for (int i = 0; i < RT; i++) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int n = wn + 32 * i + 2 * e + 4 * hh;
                    const float4 sw = *reinterpret_cast<const float4*>(side_w + n);
                    const float4 bias = *reinterpret_cast<const float4*>(side_b + n);
                    const float s4[4] = {sw.x, sw.y, sw.z, sw.w}, b4[4] = {bias.x, bias.y, bias.z, bias.w};
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        v[e + u] = finish(acc[i][j][e + u], s4[u], sx, a.bias != nullptr, b4[u]);
                }
#pragma unroll
                for (int p = 0; p < 2; p++) {  // channels 16 p + 8 hh .. + 7
                    const int n = n0 + wn + 32 * i + 16 * p + 8 * hh;
                    if constexpr (DT == TN_F32) {
                        float y[8];
#pragma unroll
                        for (int u = 0; u < 4; u++) trade(v[8 * p + u], v[8 * p + 4 + u], y[u], y[4 + u]);
                        if (m < a.m) put8(static_cast<float*>(a.y) + row + n, y, whole ? 8 : a.n - n);
                    } else {
                        using E = El<DT == TN_F16>;
                        uint32_t y[4];
#pragma unroll
                        for (int u = 0; u < 2; u++)
                            trade(E::pack_out(v[8 * p + 2 * u], v[8 * p + 2 * u + 1]),
                                  E::pack_out(v[8 * p + 4 + 2 * u], v[8 * p + 5 + 2 * u]), y[u], y[2 + u]);
                        if (m < a.m) put8(static_cast<uint16_t*>(a.y) + row + n, y, whole ? 8 : a.n - n);
                    }
                }
            }
        }
    };
    if (a.y_dtype == TN_F32) leave(std::integral_constant<int, TN_F32>{});
    else if (a.y_dtype == TN_BF16) leave(std::integral_constant<int, TN_BF16>{});
    else leave(std::integral_constant<int, TN_F16>{});
}

// Tile t of ntl x mtl: consecutive ones of a die's share; there eight token tiles at a time,
// then the next channels, so that what a die's tiles read stays in its cache.
struct Place {
    int m, n;
};
__device__ inline int of_die(int id, int count) {
    const int q = count / 8, rem = count % 8, die = id % 8;
    return die * q + min(die, rem) + id / 8;
}
__device__ inline Place place_of(int t, int ntl, int mtl) {
    constexpr int GM = 8;
    const int gsize = GM * ntl, group = t / gsize, gm = min(GM, mtl - group * GM), in = t - group * gsize;
    return {group * GM + in % gm, in / gm};
}

template <int WN, int WM, int RT, int CT, int KB, int NS, int KG = 1>
__global__ __launch_bounds__(64 * WN * WM * KG, 2) void k_i8_gemm(const MmArgs a, int ntl, int mtl, int nwg) {
    using T = Tile<WN, WM, RT, CT, KB, NS, KG>;
    __shared__ __align__(16) uint8_t ring[NS * T::STAGE];
    __shared__ __align__(16) float side[3 * T::SIDE];
    const int id = wg_number();
    if (id >= nwg) return;
    const Place p = place_of(of_die(id, nwg), ntl, mtl);
    gemm_tile<WN, WM, RT, CT, KB, NS, KG>(a, ring, side, p.m * T::BM, p.n * T::BN);
}

// Tiles of 256 x 256, one a compute unit; the last `halved` of them as two of half the
// tokens, so that a round that would leave half of the units idle takes about half as long.
// (47 registers spill, 168 bytes a lane, all in the epilogues: none in a loop over K.)
__global__ __launch_bounds__(512, 2) void k_i8_large(const MmArgs a, int ntl, int mtl, int halved) {
    using T = Tile<2, 4, 4, 2, 128, 2>;
    using H = Tile<2, 4, 4, 1, 128, 2>;
    __shared__ __align__(16) uint8_t ring[2 * T::STAGE];
    __shared__ __align__(16) float side[3 * T::SIDE];
    const int id = wg_number(), whole = ntl * mtl - halved;
    if (id < whole) {
        const Place p = place_of(of_die(id, whole), ntl, mtl);
        gemm_tile<2, 4, 4, 2, 128, 2>(a, ring, side, p.m * T::BM, p.n * T::BN);
    } else {
        const int x = id - whole;
        if (x >= 2 * halved) return;
        const int t = of_die(x, 2 * halved);
        const Place p = place_of(whole + t / 2, ntl, mtl);
        const int m0 = p.m * T::BM + t % 2 * H::BM;
        if (m0 < a.m) gemm_tile<2, 4, 4, 1, 128, 2>(a, ring, side, m0, p.n * T::BN);
    }
}

template <int WN, int WM, int RT, int CT, int KB, int NS, int KG = 1>
tn_status gemm_launch(hipStream_t st, const MmArgs& a) {
    using T = Tile<WN, WM, RT, CT, KB, NS, KG>;
    const int64_t ntl = cdiv(a.n, T::BN), mtl = cdiv(a.m, T::BM);
    if (ntl * mtl > INT32_MAX) return fail(TN_EVALUE, "i8_matmul: shape too large");
    hipLaunchKernelGGL((k_i8_gemm<WN, WM, RT, CT, KB, NS, KG>), wg_grid(ntl * mtl), dim3(64 * T::W * KG), 0, st, a, (int)ntl,
                       (int)mtl, (int)(ntl * mtl));
    TN_LAUNCHED();
    return TN_OK;
}

tn_status large_launch(hipStream_t st, const MmArgs& a) {
    const int64_t ntl = cdiv(a.n, 256), mtl = cdiv(a.m, 256), tiles = ntl * mtl;
    if (tiles + 256 > INT32_MAX) return fail(TN_EVALUE, "i8_matmul: shape too large");
    const int64_t left = tiles % 256, halved = left <= 128 ? left : 0;
    hipLaunchKernelGGL(k_i8_large, wg_grid(tiles + halved), dim3(512), 0, st, a, (int)ntl, (int)mtl, (int)halved);
    TN_LAUNCHED();
    return TN_OK;
}

// ---- few rows ------------------------------------------------------------------------
//
// A workgroup takes 16 channels of up to 16 tokens; its eight waves an eighth of K each,
// operands straight from memory, eight steps of 64 at a time, and add their sums up in
// LDS. Bound by the weights' bytes and, over few channels, by a wave's loads one behind
// the other.
constexpr int FEW_W = 8, FEW_U = 8;

struct FewSums {
    i32x4 part[FEW_W][64];
};

// The waves' sums (channels 4 g .. 4 g + 3 of token c) to the outputs.
__device__ inline void few_out(const MmArgs& a, FewSums& s, const i32x4& acc, int n0, const float* sx) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    s.part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    i32x4 t = s.part[0][lane];
#pragma unroll
    for (int i = 1; i < FEW_W; i++) t += s.part[i][lane];
    const int n = n0 + 4 * g;
    if (c >= a.m) return;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        if (n + u >= a.n) break;
        const float v = finish(t[u], a.w.s[n + u], sx[c], a.bias != nullptr, a.bias ? a.bias[n + u] : 0.0f);
        const int64_t i = (int64_t)c * a.n + n + u;
        if (a.y_dtype == TN_F32) static_cast<float*>(a.y)[i] = v;
        else static_cast<uint16_t*>(a.y)[i] = a.y_dtype == TN_BF16 ? bf16_out(v) : f16_out(v);
    }
}

// acc += the products of N steps from step k on.
template <int N>
__device__ __attribute__((always_inline)) inline void few_steps(const int8_t* px, const int8_t* pw, int k, i32x4& acc) {
    i32x4 x[N], w[N];
#pragma unroll
    for (int u = 0; u < N; u++) w[u] = *reinterpret_cast<const i32x4*>(pw + 64 * (k + u));
#pragma unroll
    for (int u = 0; u < N; u++) x[u] = *reinterpret_cast<const i32x4*>(px + 64 * (k + u));
#pragma unroll
    for (int u = 0; u < N; u++) acc = mfma_i8(w[u], x[u], acc);
}

__global__ __launch_bounds__(64 * FEW_W) void k_i8_few(const MmArgs a) {
    __shared__ FewSums sums;
    __shared__ float sx[16];
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16;
    if (threadIdx.x < 16) sx[threadIdx.x] = a.a.s[min((int)threadIdx.x, a.m - 1)];
    const int8_t* px = a.a.c + (int64_t)min(c, a.m - 1) * a.pitch + 16 * g;
    const int8_t* pw = a.w.c + (int64_t)min(n0 + c, a.n - 1) * a.pitch + 16 * g;
    i32x4 acc = {0, 0, 0, 0};
    const int steps = a.pitch / 64, hi = (int)((int64_t)steps * (wave + 1) / FEW_W);
    int k = (int)((int64_t)steps * wave / FEW_W);
    for (; k + FEW_U <= hi; k += FEW_U) few_steps<FEW_U>(px, pw, k, acc);
    for (; k < hi; k++) few_steps<1>(px, pw, k, acc);
    few_out(a, sums, acc, n0, sx);
}

// The same on rows as they are, up to FUSED_M of them: every workgroup quantises them into
// LDS, its first weights on their way meanwhile. Saves the prepass's launch. us of one and of
// four bf16 rows: [4096, 4096] 5.4 and 8.0, [14336, 4096] 15.3 and 18.9 (sixteen, quantised
// ahead and in tiles, 14.9: over many channels the rule, which does not ask for them, is late).
constexpr int FUSED_M = 4;
constexpr int64_t FUSED_BYTES = 32 << 10;  // of codes

template <int DT>
__global__ __launch_bounds__(64 * FEW_W) void k_i8_fused(const MmArgs a, const void* __restrict__ x, int k_len) {
    __shared__ __align__(16) int8_t codes[FUSED_BYTES];
    __shared__ FewSums sums;
    __shared__ float sx[16], red[FEW_W];
    __shared__ int bad[FEW_W];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 16;
    const int8_t* pw = a.w.c + (int64_t)min(n0 + c, a.n - 1) * a.pitch + 16 * g;
    const int steps = a.pitch / 64, hi = (int)((int64_t)steps * (wave + 1) / FEW_W);
    int k = (int)((int64_t)steps * wave / FEW_W);
    i32x4 w[FEW_U];
#pragma unroll
    for (int u = 0; u < FEW_U; u++) w[u] = *reinterpret_cast<const i32x4*>(pw + 64 * min(k + u, steps - 1));
    for (int r = 0; r < a.m; r++) {
        const int64_t at = (int64_t)r * k_len;
        Eight<DT> v;
        float top = 0.0f, nan = 0.0f;
        load_row8<DT>(x, at, 8 * tid, k_len, v);
        measure(v, top, nan);
        for (int i = 8 * (64 * FEW_W + tid); i < k_len; i += 8 * 64 * FEW_W) {
            Eight<DT> y;
            load_row8<DT>(x, at, i, k_len, y);
            measure(y, top, nan);
        }
        top = xor32_max(xor16_max(row16_max(top)));
        bool odd = __any(nan != nan);
        if (lane == 0) red[wave] = top, bad[wave] = odd;
        __syncthreads();
        odd = false;
#pragma unroll
        for (int i = 0; i < FEW_W; i++) top = fmaxf(top, red[i]), odd |= bad[i] != 0;
        const float s = scale_of(top), inv = s > 0.0f ? 1.0f / s : 0.0f;
        if (tid == 0) sx[r] = odd ? NAN : s;
        int8_t* out = codes + r * a.pitch;
        if (8 * tid < a.pitch) *reinterpret_cast<uint2*>(out + 8 * tid) = codes8(v, inv, odd);
        for (int i = 8 * (64 * FEW_W + tid); i < a.pitch; i += 8 * 64 * FEW_W) {
            Eight<DT> y;
            load_row8<DT>(x, at, i, k_len, y);
            *reinterpret_cast<uint2*>(out + i) = codes8(y, inv, odd);
        }
        __syncthreads();
    }
    const int8_t* px = codes + min(c, a.m - 1) * a.pitch + 16 * g;
    i32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < FEW_U; u++)
        if (k + u < hi) acc = mfma_i8(w[u], *reinterpret_cast<const i32x4*>(px + 64 * (k + u)), acc);
    k += FEW_U;
    for (; k + FEW_U <= hi; k += FEW_U) few_steps<FEW_U>(px, pw, k, acc);
    for (; k < hi; k++) few_steps<1>(px, pw, k, acc);
    few_out(a, sums, acc, n0, sx);
}

bool fused(int64_t m, int64_t k) { return m <= FUSED_M && m * pitch_of(k) <= FUSED_BYTES; }

tn_status few_launch(hipStream_t st, const MmArgs& a) {
    hipLaunchKernelGGL(k_i8_few, dim3((unsigned)cdiv(a.n, 16)), dim3(64 * FEW_W), 0, st, a);
    TN_LAUNCHED();
    return TN_OK;
}

tn_status fused_launch(hipStream_t st, const MmArgs& a, const void* x, int dtype, int64_t k) {
    const dim3 grid((unsigned)cdiv(a.n, 16)), block(64 * FEW_W);  // n < 2^24: fewer than 2^30 threads
    if (dtype == TN_F32) hipLaunchKernelGGL(k_i8_fused<TN_F32>, grid, block, 0, st, a, x, (int)k);
    else if (dtype == TN_BF16) hipLaunchKernelGGL(k_i8_fused<TN_BF16>, grid, block, 0, st, a, x, (int)k);
    else hipLaunchKernelGGL(k_i8_fused<TN_F16>, grid, block, 0, st, a, x, (int)k);
    TN_LAUNCHED();
    return TN_OK;
}

// The tile shapes, by what a call takes in rounds of the workgroups that the 256 units
// hold: us of a round over K = 4096 with one and with two workgroups a unit (it holds one
// where both are the same), and of a tile's start and end, both fitted to measurements of
// 1 to 4096 tokens on six weights. (us at the best shape, and at its neighbours; [m, 4096]
// x [14336, 4096] where not stated: m 32, 64 x 32 13.8, 64 x 64 15.3; m 64, 64 x 64 of two
// groups 15.2, 64 x 128 18.2; m 128, 64 x 128 of two groups 19.3, 64 x 64 22.9; m 512, 128 x
// 128 40.8, 64 x 128 53, 256 x 256 45; m 1024, 256 x 256 73, 128 x 128 79. [64, 4096] x
// [4096, 4096]: 64 x 32 7.9, 64 x 64 9.3, of one group 11.4; [256, 14336] x [4096, 14336]: 64
// x 64 34.7, 64 x 128 47.8, 128 x 128 97.)
struct Shape {
    int bn, bm;
    float one, two, ends;
    tn_status (*launch)(hipStream_t, const MmArgs&);
};
const Shape SHAPES[] = {
    {64, 32, 5.3f, 5.3f, 0.6f, gemm_launch<2, 1, 1, 1, 128, 3, 4>},
    {64, 64, 7.2f, 7.2f, 0.7f, gemm_launch<2, 2, 1, 1, 128, 3, 2>},
    {64, 64, 9.5f, 14.0f, 0.7f, gemm_launch<2, 2, 1, 1, 128, 4>},
    {64, 128, 11.8f, 11.8f, 1.2f, gemm_launch<2, 2, 1, 2, 128, 3, 2>},
    {64, 128, 13.5f, 23.0f, 1.0f, gemm_launch<2, 2, 1, 2, 128, 3>},
    {128, 128, 24.0f, 38.0f, 2.3f, gemm_launch<2, 2, 2, 2, 128, 2>},
    {256, 256, 36.5f, 66.0f, 4.5f, large_launch},
};

tn_status matmul(hipStream_t st, const MmArgs& a) {
    // (us, here and in tiles of 64 x 32: 16 tokens of [4096, 4096], 7.1 and 7.5, of [4096,
    // 14336], 17.9 and 24.9, of [5000, 1536], 6.0 and 5.4, of [14336, 4096], 19.8 and 13.5)
    if (a.m <= 16 && a.n <= 8192) return few_launch(st, a);
    const Shape* best = SHAPES;
    double least = INFINITY;
    for (const Shape& s : SHAPES) {
        const int64_t tiles = cdiv(a.n, s.bn) * cdiv(a.m, s.bm);
        const bool large = s.launch == large_launch;  // (its tiles of half the tokens: the short round)
        const int64_t slots = s.one == s.two || large ? 256 : 512, rest = tiles % slots;
        const int64_t rounds = cdiv(tiles, slots);
        double us = (double)(tiles / slots) * s.two;
        if (rest) us += rest <= (large ? 128 : 256) ? s.one : s.two;
        us = us * a.pitch / 4096 + (double)rounds * s.ends;
        if (us < least) least = us, best = &s;
    }
    return best->launch(st, a);
}

template <int DT>
void rows_launch(hipStream_t st, const void* x, int m, int k, int8_t* codes, float* scales) {
    const dim3 waves((unsigned)cdiv(m, 4)), rows((unsigned)m);
    if (k <= 2048) hipLaunchKernelGGL((k_i8_rows<DT, 64, 4>), waves, dim3(256), 0, st, x, m, k, codes, scales);
    else if (k <= 4096)
        hipLaunchKernelGGL((k_i8_rows<DT, 64, 8>), waves, dim3(256), 0, st, x, m, k, codes, scales);
    else hipLaunchKernelGGL((k_i8_rows<DT, 256, 4>), rows, dim3(256), 0, st, x, m, k, codes, scales);
}

tn_status quantize(hipStream_t st, const void* x, int dtype, int64_t m, int64_t k, int8_t* codes, float* scales) {
    if (dtype == TN_F32) rows_launch<TN_F32>(st, x, (int)m, (int)k, codes, scales);
    else if (dtype == TN_BF16) rows_launch<TN_BF16>(st, x, (int)m, (int)k, codes, scales);
    else rows_launch<TN_F16>(st, x, (int)m, (int)k, codes, scales);
    TN_LAUNCHED();
    return TN_OK;
}

bool row_dtype(int dtype) { return dtype == TN_F32 || dtype == TN_BF16 || dtype == TN_F16; }
bool unaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }
int64_t size_of(int dtype) { return dtype == TN_F32 ? 4 : 2; }
// Whether y [m, n] and `bytes` bytes at p have any in common: a product writes y while others of
// its workgroups read.
bool overlaps(const void* y, int64_t m, int64_t n, int y_dtype, const void* p, int64_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(y), b = reinterpret_cast<uintptr_t>(p);
    return a < b + (uintptr_t)bytes && b < a + (uintptr_t)(m * n * size_of(y_dtype));
}

tn_status size_check(const char* op, int64_t m, int64_t k, int64_t n) {
    if (k <= 0)
        return fail(TN_EINVAL, std::string(op) + ": mat1 and mat2 shapes cannot be multiplied ([" + std::to_string(m) +
                                   ", " + std::to_string(k) + "] and " + std::to_string(k) + "x" + std::to_string(n) + ")");
    if (m < 0 || n < 0) return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    if (k > MAX_K)
        return fail(TN_ENOTIMPL, std::string(op) + ": " + std::to_string(k) + " elements a row; at most " +
                                     std::to_string(MAX_K) + " are implemented");
    if (m > MAX_ROWS || n > MAX_ROWS) return fail(TN_EVALUE, std::string(op) + ": shape too large");
    return TN_OK;
}

int64_t work_bytes(int64_t m, int64_t k) { return fused(m, k) ? 0 : m * pitch_of(k) + (m * 4 + 15) / 16 * 16; }

}  // namespace
}  // namespace tn

using namespace tn;

extern "C" {

int64_t tn_i8_pitch(int64_t k) { return k > 0 ? pitch_of(k) : 0; }

tn_status tn_i8_quantize(void* stream, const void* x, int dtype, int64_t m, int64_t k, int8_t* codes, float* scales) {
    const char* op = "i8_quantize";
    if (!row_dtype(dtype)) return fail(TN_ENOTIMPL, "i8_quantize: rows must be float32, bfloat16 or float16");
    TN_TRY(size_check(op, m, k, 0));
    if (m == 0) return TN_OK;
    if (!x || !codes || !scales) return fail(TN_EVALUE, "i8_quantize: null pointer");
    if (unaligned(codes)) return fail(TN_EVALUE, "i8_quantize: codes must be 16-byte aligned");
    return quantize((hipStream_t)stream, x, dtype, m, k, codes, scales);
}

tn_status tn_i8_matmul(void* stream, const int8_t* a, const float* a_scales, int64_t m, int64_t k, const int8_t* w,
                       const float* w_scales, int64_t n, const float* bias, void* y, int y_dtype) {
    const char* op = "i8_matmul";
    if (!row_dtype(y_dtype)) return fail(TN_ENOTIMPL, "i8_matmul: the output must be float32, bfloat16 or float16");
    TN_TRY(size_check(op, m, k, n));
    if (m == 0 || n == 0) return TN_OK;
    if (!a || !a_scales || !w || !w_scales || !y) return fail(TN_EVALUE, "i8_matmul: null pointer");
    if (unaligned(a) || unaligned(w)) return fail(TN_EVALUE, "i8_matmul: codes must be 16-byte aligned");
    if (overlaps(y, m, n, y_dtype, a, m * pitch_of(k)) || overlaps(y, m, n, y_dtype, w, n * pitch_of(k)))
        return fail(TN_EINVAL, "i8_matmul: y overlaps an input");
    MmArgs p{{a, a_scales}, {w, w_scales}, bias, y, (int)m, (int)n, (int)pitch_of(k), y_dtype};
    return matmul((hipStream_t)stream, p);
}

int64_t tn_i8_linear_work_bytes(int64_t m, int64_t k) {
    if (size_check("i8_linear_work_bytes", m, k, 0) != TN_OK) return 0;
    return work_bytes(m, k);
}

tn_status tn_i8_linear(void* stream, const void* x, int x_dtype, int64_t m, int64_t k, const int8_t* w,
                       const float* w_scales, int64_t n, const float* bias, void* work, int64_t work_size, void* y,
                       int y_dtype) {
    const char* op = "i8_linear";
    if (!row_dtype(x_dtype)) return fail(TN_ENOTIMPL, "i8_linear: the activation must be float32, bfloat16 or float16");
    if (!row_dtype(y_dtype)) return fail(TN_ENOTIMPL, "i8_linear: the output must be float32, bfloat16 or float16");
    TN_TRY(size_check(op, m, k, n));
    if (m == 0 || n == 0) return TN_OK;
    const int64_t need = tn_i8_linear_work_bytes(m, k);
    if (work_size < need)
        return fail(TN_EVALUE, "i8_linear: work holds " + std::to_string(work_size) + " bytes, this call needs " +
                                   std::to_string(need));
    if (!x || !w || !w_scales || !y || (need && !work)) return fail(TN_EVALUE, "i8_linear: null pointer");
    if (unaligned(w) || (need && unaligned(work))) return fail(TN_EVALUE, "i8_linear: codes and work must be 16-byte aligned");
    if (overlaps(y, m, n, y_dtype, x, m * k * size_of(x_dtype)) || overlaps(y, m, n, y_dtype, w, n * pitch_of(k)) ||
        overlaps(y, m, n, y_dtype, work, need))
        return fail(TN_EINVAL, "i8_linear: y overlaps an input or work");
    if (fused(m, k)) {
        const MmArgs p{{nullptr, nullptr}, {w, w_scales}, bias, y, (int)m, (int)n, (int)pitch_of(k), y_dtype};
        return fused_launch((hipStream_t)stream, p, x, x_dtype, k);
    }
    int8_t* codes = static_cast<int8_t*>(work);
    float* scales = reinterpret_cast<float*>(codes + m * pitch_of(k));
    const Turn turn(stream);
    TN_TRY(quantize((hipStream_t)stream, x, x_dtype, m, k, codes, scales));
    MmArgs p{{codes, scales}, {w, w_scales}, bias, y, (int)m, (int)n, (int)pitch_of(k), y_dtype};
    return matmul((hipStream_t)stream, p);
}

}  // extern "C"
