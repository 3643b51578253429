// Attention of ragged rows over the paged 8-bit cache (tnhip.h describes the
// planes and the rows).
//
// Rows of a request are folded over the query heads that share a key/value head:
// row i of (request, key/value head) is token i / G, head h * G + i % G, so that
// G heads read each key once. Scores are computed transposed, S^T = K Q^T, and so
// is the output, O^T = V^T P^T: the lane that holds a column's scores then holds
// them as P^T's operand, with no exchange between lanes (below).
//
// A byte under the bits of f16's 1024 is 1024 + byte, and 1152 less its code: two
// instructions a pair, exact. So codes enter both products exactly, and the scales,
// one for sixteen keys, are applied to scores and to probabilities.
#include "paged_rows.h"

#include <algorithm>
#include <cmath>

namespace tn {
namespace {

using Paged8Args = Ragged<Pages8>;

// A row's part of a split: its sums, then the running maximum, the sum of
// probabilities and the scale of its values (Vref), in four floats.
struct Part {
    float m, l, v, pad;
};

// Parts of each 16-bit operand: a 16-bit query is one f16 (a bf16 row scaled by a power
// of two), an f32 one two. Probabilities are one for bf16 rows, where half a step of f16 is
// an eighth of the output's own, and two for others: in one, f16 rows would be off by about
// as much again as their rounding (2.9e-4 of the output's norm in place of 2.1e-4). us, in
// two parts / in one, f16: a prompt of 4096 of 32/8 heads of 128 elements 203 / 160, 512 rows
// behind 4096 75 / 65, six ragged requests of 16/4 heads of 64 50 / 44, sixteen single
// tokens over 512 to 4096 21.8 / 20.9, twelve over 20000 to 40000 138 / 136.
template <int DT>
struct Parts8 {
    static constexpr int Q = DT == TN_F32 ? 2 : 1, P = DT == TN_BF16 ? 1 : 2;
};

// Eight codes of two dwords as f16, exactly.
TN_INLINE h8 codes8(uint32_t a, uint32_t b) {
#if __HIP_DEVICE_COMPILE__
    const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    auto pk_sum = [](uint32_t x, h2 y) { return __builtin_bit_cast(uint32_t, as_h2(x) + y); };
    auto low = [&](uint32_t w) { return pk_sum(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u), off); };
    auto high = [&](uint32_t w) { return pk_sum(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u), off); };
    return as_h8(low(a), high(a), low(b), high(b));
#else
    (void)a, (void)b;
    return h8{};
#endif
}

// The scale of values that a row's sums are held under: a power of two above the scale of every
// block met so far that the row attends, so that a probability times its block's share of it is at
// most itself, and no later token's values take part.
TN_INLINE float vref_for(float scale) {
    const uint32_t e = (__builtin_bit_cast(uint32_t, scale) >> 23) & 0xffu;
    return __builtin_bit_cast(float, min(e + 1u, 253u) << 23);
}
// Over the two or four lanes of a quad.
template <int N>
TN_INLINE float quad_max(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    if constexpr (N == 4) v = fmaxf(v, dpp_f<0x4E>(v));
    return v;
}
constexpr float VREF_MIN = 1.1754943508222875e-38f;  // 2^-126
// Its inverse, exactly.
TN_INLINE float vref_inverse(float vref) {
    return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, vref));
}

// ---- few rows ---------------------------------------------------------------------
//
// A wave takes 64 keys at a time, four blocks. Tile t (0 .. 3) of S^T has keys
// 16 g + 4 t + i in row 4 g + i (lane c + 16 g holds rows 4 g .. 4 g + 3 of column c),
// so that a lane holds the sixteen keys of one block, whose scales are one number each
// for keys and for values, and the operands of its part of two 32-key products
// O^T += V^T P^T, whose values it reads as sixteen bytes a column.
//
// A wave works alone, on every fourth (times the splits) run of tiles, the next tile's codes in
// registers while one is computed, which is what a call of single tokens is bound by: twelve f16
// tokens over 20000 to 40000 keys, 32/8 heads of 128 elements, 737 MB, 138 us, 5.3 TB/s; sixteen
// bf16 over 512 to 4096 22 us (76 MB, 18 us of it here, the rest its merge's).
template <int NB>
struct KeyTile8 {
    uint32_t k[4][2 * NB];  // this lane's part of a row of each score tile
    uint32_t v[2 * NB][4];  // its block's values, a column of each sixteen elements
    float ks, vs;           // its block's scales
    int bad;                // its block's page is outside the cache
};

template <int DT, int NB>
__global__ __launch_bounds__(256, (NB <= 4 ? 2 : 1)) void k_paged8_few(const Paged8Args a) {
    constexpr int PQ = Parts8<DT>::Q, PP = Parts8<DT>::P, D = 32 * NB, W2 = NB / 2;
    __shared__ __align__(16) float so[4][16][D + 4];
    __shared__ Part sml[4][16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int r = blockIdx.z, h = (int)blockIdx.y % a.c.H, first = (int)blockIdx.y / a.c.H * 16;
    const int start = start_of(a, r), all = rows_of(a, r, start);
    const int c = min(all, a.max_rows), rows = c * a.G;
    if (first >= rows || rows > a.few) return;
    const int len = max(0, min(a.lens[r], a.max_len));
    const int S = 1 << a.c.shift;
    // this lane's column: its row, and the keys it attends
    const int i = first + col, j = min(i, rows - 1) / a.G;
    const int hq = h * a.G + min(i, rows - 1) % a.G;
    const int keys = max(0, len - all + j + 1);
    const int most = max(0, len - all + (min(first + 16, rows) - 1) / a.G + 1);  // of any row
    const int least = max(0, len - all + first / a.G + 1);                       // of every row

    // The query as f16 parts: product b contracts over the eight elements of each lane
    // group that the codes' loads give it.
    h8 q[PQ][NB];
    float rs = fabsf(a.sl2);
    {
        float x[NB][8], top = 0.0f;
        const int64_t qi = (int64_t)(start + j) * a.q_stride + (int64_t)hq * D;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            Eight<DT> e8;
            e8.load(a.q, qi + (b < 2 * W2 ? 64 * (b >> 1) + 16 * g + 8 * (b & 1) : 32 * b + 8 * g));
#pragma unroll
            for (int e = 0; e < 8; e++) x[b][e] = e8.get(e), top = fmaxf(top, fabsf(x[b][e]));
        }
        float sc = 1.0f;
        if constexpr (DT != TN_F16) {
            sc = row_scale(wave_xor_max(top));
            rs = rs / sc;
        }
        // a positive factor, so that it can be taken out of the maximum
        rs = fmaxf(rs, 1.1754944e-38f);
        if (a.sl2 < 0.0f) sc = -sc;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = x[b][e] * sc;
                const _Float16 hi = (_Float16)v;
                q[0][b][e] = hi;
                if constexpr (PQ == 2) q[1][b][e] = (_Float16)(v - (float)hi);
            }
    }

    f32x4 o[2 * NB];
#pragma unroll
    for (int t = 0; t < 2 * NB; t++) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f, vref = VREF_MIN;

    // this wave's tiles
    const int nt = (most + 63) >> 6, nw = a.nsplit * 4, gw = (int)blockIdx.x * 4 + w;
    const int lo = (int)((int64_t)gw * nt / nw), hi = (int)((int64_t)(gw + 1) * nt / nw);
    const int32_t* table = a.table + (int64_t)r * a.width;
    // the pages of the block whose key rows this lane reads, and of its own
    auto pages = [&](int t) __attribute__((always_inline)) {
        const int last = a.width - 1;
        return make_int2(table[min((64 * t + 16 * (col >> 2)) >> a.c.shift, last)],
                         table[min((64 * t + 16 * g) >> a.c.shift, last)]);
    };
    auto load = [&](KeyTile8<NB>& x, int t, int2 pg) __attribute__((always_inline)) {
        const bool bk = (unsigned)pg.x >= (unsigned)a.c.pages, bv = (unsigned)pg.y >= (unsigned)a.c.pages;
        const int64_t rk = (((int64_t)(bk ? 0 : pg.x) * a.c.H + h) << a.c.shift) + ((64 * t + 16 * (col >> 2)) & (S - 1));
        const int64_t rv = (((int64_t)(bv ? 0 : pg.y) * a.c.H + h) << a.c.shift) + ((64 * t + 16 * g) & (S - 1));
        const uint8_t* pk = a.c.kc + (rk + (col & 3)) * D;
        x.bad = bv;
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int s = 0; s < W2; s++) {
                uint32_t y[4];
                load_words(pk + 4 * u * D + 64 * s + 16 * g, y);
#pragma unroll
                for (int e = 0; e < 4; e++) x.k[u][4 * s + e] = y[e];
            }
            if constexpr (NB % 2) {
                uint32_t y[2];
                load_words(pk + 4 * u * D + 64 * W2 + 8 * g, y);
                x.k[u][4 * W2] = y[0], x.k[u][4 * W2 + 1] = y[1];
            }
        }
        const uint8_t* pv = a.c.vc + rv * D + col * 16;
#pragma unroll
        for (int b = 0; b < 2 * NB; b++) load_words(pv + 256 * b, x.v[b]);
        x.ks = a.c.ks[rv >> 4], x.vs = a.c.vs[rv >> 4];
    };
    auto compute = [&](KeyTile8<NB>& x, int t) __attribute__((always_inline)) {
        f32x4 s[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            s[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const h8 kf = codes8(x.k[u][2 * b], x.k[u][2 * b + 1]);
                if constexpr (PQ == 2) s[u] = mfma16(kf, q[1][b], s[u]);
                s[u] = mfma16(kf, q[0][b], s[u]);
            }
        }
        const int k0 = 64 * t + 16 * g;
        const bool edge = 64 * t + 64 > least || __any(x.bad);
        const float f = rs * x.ks;
#pragma unroll
        for (int u = 0; u < 4; u++) s[u] = s[u] * f;
        if (edge) {
            // values of a block that this lane's row does not attend count as zeros, whatever its page
            // holds, so that the reference for the scales is of the row's own keys
            if (k0 >= keys || x.bad) x.vs = 0.0f;
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = s[u][e];
                    s[u][e] = k0 + 4 * u + e >= keys ? -INFINITY : x.bad ? NAN : v;
                }
        }
        const float mx = wave_xor_max(
            max3f(max3f(max3f(s[0][0], s[0][1], s[0][2]), max3f(s[0][3], s[1][0], s[1][1]), s[1][2]),
                  max3f(max3f(s[1][3], s[2][0], s[2][1]), max3f(s[2][2], s[2][3], s[3][0]), s[3][1]),
                  fmaxf(s[3][2], s[3][3])));
        if (__any(mx > m + RESCALE_SLACK)) {
            const float mn = fmaxf(m, mx), al = exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) o[b] = o[b] * al;
        }
        const float mv = wave_xor_max(x.vs);
        if (__any(mv >= vref)) {
            const float nv = mv >= vref ? vref_for(mv) : vref, al = vref * vref_inverse(nv);
            vref = nv;
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) o[b] = o[b] * al;
        }
        const float mu = P_BIAS - (m == -INFINITY ? 0.0f : m), share = x.vs * vref_inverse(vref);
        uint32_t ph[8], pl[8];
#pragma unroll
        for (int n = 0; n < 16; n += 2) {
            const float p0 = __builtin_amdgcn_exp2f(s[n >> 2][n & 3] + mu);
            const float p1 = __builtin_amdgcn_exp2f(s[n >> 2][(n & 3) + 1] + mu);
            l += p0;
            l += p1;
            float none = 0.0f;
            split_p<PP>(p0 * share, p1 * share, ph[n >> 1], pl[n >> 1], none);
        }
#pragma unroll
        for (int b = 0; b < 2 * NB; b++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const h8 vf = codes8(x.v[b][2 * u], x.v[b][2 * u + 1]);
                if constexpr (PP == 2)
                    o[b] = mfma16(vf, as_h8(pl[4 * u], pl[4 * u + 1], pl[4 * u + 2], pl[4 * u + 3]), o[b]);
                o[b] = mfma16(vf, as_h8(ph[4 * u], ph[4 * u + 1], ph[4 * u + 2], ph[4 * u + 3]), o[b]);
            }
    };
    // the next tile on its way while one is computed, its pages before that
    if (lo < hi) {
        KeyTile8<NB> x, y;
        int2 pg = pages(lo), next = pages(min(lo + 1, hi - 1));
        load(x, lo, pg);
        for (int t = lo; t < hi; t += 2) {
            pg = pages(min(t + 2, hi - 1));
            load(y, min(t + 1, hi - 1), next);
            compute(x, t);
            if (t + 1 >= hi) break;
            next = pages(min(t + 3, hi - 1));
            load(x, min(t + 2, hi - 1), pg);
            compute(y, t + 1);
        }
    }

    // merge the waves
    l = wave_xor_sum(l);
    if (g == 0) sml[w][col] = Part{m, l, vref, 0.0f};
#pragma unroll
    for (int t = 0; t < 2 * NB; t++) *reinterpret_cast<f32x4*>(&so[w][col][16 * t + 4 * g]) = o[t];
    __syncthreads();
    for (int e = tid; e < 16 * (D / 4); e += 256) {
        const int rc = e / (D / 4), d = e % (D / 4) * 4, ri = first + rc;
        if (ri >= rows) break;
        float mm = -INFINITY, vv = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; s++) mm = fmaxf(mm, sml[s][rc].m), vv = fmaxf(vv, sml[s][rc].v);
        const float mu = mm == -INFINITY ? 0.0f : mm;
        float tl = 0.0f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const Part p = sml[s][rc];
            const float f = exp2f(p.m - mu), fv = f * (p.v / vv);
            tl += p.l * f;
            const f32x4 v = *reinterpret_cast<const f32x4*>(&so[s][rc][d]);
#pragma unroll
            for (int n = 0; n < 4; n++) acc[n] += v[n] * fv;
        }
        if (a.nsplit == 1) {
            const int64_t row = (int64_t)(start + ri / a.G) * a.Hq + h * a.G + ri % a.G;
            const float inv = 1.0f / tl;
            const float y[4] = {acc[0] * inv * vv, acc[1] * inv * vv, acc[2] * inv * vv, acc[3] * inv * vv};
            store4<DT>(a.out, row * D + d, y);
            if (a.lse && d == 0) a.lse[row] = tl == 0.0f ? -INFINITY : (mm - P_BIAS) * LN2 + logf(tl);
        } else {
            const int64_t row = (((int64_t)r * a.c.H + h) * a.few + ri) * a.nsplit + blockIdx.x;
            *reinterpret_cast<f32x4*>(a.part_o + row * D + d) = acc;
            if (d == 0) reinterpret_cast<Part*>(a.part_ml)[row] = Part{mm, tl, vv, 0.0f};
        }
    }
}

// Splits of a row, in order (the same bits every time), into four output columns of a row of
// `out`, -1: none, which row_of() tells. Every load of up to JOINS splits is on its way before
// anything waits for one; one wave or few a compute unit, so that is what the time goes by.
constexpr int JOINS = 8;
template <int DT, class RowOf>
TN_INLINE void join(const Paged8Args& a, const float* po, const Part* ml, int ns, int d, RowOf row_of) {
    const int D = 32 * a.c.nb;
    f32x4 v[JOINS];
    Part p[JOINS];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < JOINS; s++) {
            const int at = min(s0 + s, ns - 1);
            p[s] = ml[at];
            v[s] = *reinterpret_cast<const f32x4*>(po + (int64_t)at * D);
        }
    };
    load(0);
    const int64_t row = row_of();
    if (row < 0) return;
    float mm = -INFINITY, tl = 0.0f, vv = 0.0f;
#pragma unroll
    for (int s = 0; s < JOINS; s++) mm = fmaxf(mm, p[s].m), vv = fmaxf(vv, p[s].v);  // (the last more than once)
    for (int s = JOINS; s < ns; s++) mm = fmaxf(mm, ml[s].m), vv = fmaxf(vv, ml[s].v);
    const float mu = mm == -INFINITY ? 0.0f : mm;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0;;) {
#pragma unroll
        for (int s = 0; s < JOINS; s++) {
            if (s0 + s >= ns) break;
            const float f = exp2f(p[s].m - mu), fv = f * (p[s].v / vv);
            tl += p[s].l * f;
#pragma unroll
            for (int n = 0; n < 4; n++) acc[n] += v[s][n] * fv;
        }
        if ((s0 += JOINS) >= ns) break;
        load(s0);
    }
    const float inv = 1.0f / tl;
    const float y[4] = {acc[0] * inv * vv, acc[1] * inv * vv, acc[2] * inv * vv, acc[3] * inv * vv};
    store4<DT>(a.out, row * D + d, y);
    if (a.lse && d == 0) a.lse[row] = tl == 0.0f ? -INFINITY : (mm - P_BIAS) * LN2 + logf(tl);
}

template <int DT>
__global__ __launch_bounds__(64) void k_paged8_combine(const Paged8Args a) {
    const int D = 32 * a.c.nb, q4 = D / 4, h = blockIdx.y, r = blockIdx.z;
    const uint32_t e = blockIdx.x * 64 + threadIdx.x;
    const int i = (int)(e / (uint32_t)q4), d = (int)(e - (uint32_t)(i * q4)) * 4;
    if (i >= a.few) return;
    const int64_t part = (((int64_t)r * a.c.H + h) * a.few + i) * a.nsplit;
    join<DT>(a, a.part_o + part * D + d, reinterpret_cast<const Part*>(a.part_ml) + part, a.nsplit, d, [&]() {
        const int start = start_of(a, r), c = min(rows_of(a, r, start), a.max_rows);
        if (i >= c * a.G || c * a.G > a.few) return (int64_t)-1;
        return (int64_t)(start + i / a.G) * a.Hq + h * a.G + i % a.G;
    });
}

// ---- many rows --------------------------------------------------------------------
//
// A wave takes 32 folded rows, a workgroup 128 of them, and keys KT at a time. The
// codes are unpacked to f16 once a workgroup, into LDS, ahead of their use: K as rows of
// D elements, V transposed, a row an element with its keys in the order in which the score
// product leaves them in a lane (keys 4 h .. 4 h + 3 of each eight in half h of the wave),
// so that P^T needs no exchange. Codes are exact there in one part; a score tile's rows 0
// .. 15 and 16 .. 31 are a block each, whose scales the softmax takes in: keys' in the
// factor that its argument has anyway, values' in its exponent, and out of the sum again
// (in tiles that end among a wave's rows, of small scales, and of f32 rows: by a product).
// Rows are padded by 16 bytes, which spreads 16 rows' reads over all banks.
//
// A wave alternates between two phases: the softmax of tile t; and the products, O^T +=
// V^T P^T of tile t and S^T of tile t + 1, with its share of the unpacking (V of tile
// t + 1, K of t + 2) in their shadow. A compute unit holds two workgroups, whose phases
// fall beside one another's by themselves: one of 256 rows in two groups held half a turn
// apart unpacks half as often and took as long (4096 bf16 rows of 32/8 heads of 128
// elements took the same; 2048 f32 rows 101 us against 93). With one barrier a turn two
// tiles of each in LDS suffice: behind barrier t, V(t) and K(t + 1) are read, V(t + 1) and
// K(t + 2) written, in the places of V(t - 1) and K(t), last read before it. What the
// softmax takes of a tile's scales is written two turns ahead of it, by lanes of the last
// wave, into one of four places.
//
// 4096 causal bf16 rows as above, 137 GFLOP, 155 to 171 us: 803 to 884 TFLOP/s; an f16
// product of 16384 reaches 1263. By its counters a SIMD issues vector instructions in 58 % of
// the cycles, the softmax's and the unpacking's for the most part, and its matrix core is busy
// in 41 %: the two phases all but take turns. LDS is busy in 35 %; as each fragment of 16-bit
// rows read from it feeds one product, it would be at its limit soon after if the matrix core
// were busy throughout. Spilled registers: one of f32 rows of 160 elements, outside the loop.
constexpr int MANY_ROWS = 128;  // folded rows of a workgroup
template <int DT, int NB>
struct Many8 {
    static constexpr int Q = Parts8<DT>::Q, P = Parts8<DT>::P;
    static constexpr int D = 32 * NB, KT = NB <= 4 ? 64 : 32;  // keys of a tile
    static constexpr int BL = KT / 16, WPB = 4 / BL;           // its blocks, waves that unpack one
    static constexpr int KP = 2 * D + 16, VP = 2 * KT + 16;    // row pitches, bytes
    static constexpr int KB = KT * KP, VB = D * VP, STAGE = KB + VB;
    static constexpr int N = (NB + 2 * WPB - 1) / (2 * WPB);   // 16-byte pieces a thread, of K and of V
    static constexpr int OP = (NB < 4 ? D : 128) * 4 + 16;     // row pitch on the way out
    static constexpr int LDS_BYTES = 2 * STAGE > MANY_ROWS * OP ? 2 * STAGE : MANY_ROWS * OP;
    // waves a SIMD: one where two do not have the registers
    static constexpr int WAVES = NB > (DT == TN_F32 ? 5 : 6) ? 1 : 2;
};

// A tile's scales: of its keys and of its values; of the latter, for tiles that all of a wave's 16-bit
// rows attend whole, a block's share of the reference as its logarithm and inverse (small: one is
// under 2^-6, and probabilities are multiplied by shares instead, where a scale of 0 needs none);
// the reference's last step and the reference.
struct Scales {
    float ks[4], vs[4], log[4], inv[4];
    float step, vref;
    int small, pad;
};
constexpr float LEAST_SHARE = 0x1p-6f;

// What a kernel only reads, through the scalar cache where its address is the wave's.
template <class T>
TN_INLINE T scalar(const T* p) {
#if __HIP_DEVICE_COMPILE__
    return *(const __attribute__((address_space(4))) T*)reinterpret_cast<uintptr_t>(p);
#else
    return *p;
#endif
}

// Rows first .. first + MANY_ROWS of request r, whose rows start at `start` and attend
// `before` keys more than there are rows ahead of them.
template <int DT, int NB>
TN_INLINE void many8_tile(const Paged8Args& a, uint8_t* lds, Scales* scales, int h, int r, int start, int rows, int first,
                          int len, int before) {
    using M = Many8<DT, NB>;
    constexpr int KT = M::KT, D = M::D, ROWS = MANY_ROWS, N = M::N, BL = M::BL, WPB = M::WPB;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hh = lane >> 5;
    const int S = 1 << a.c.shift;
    const int i = first + 32 * w + col, j = min(i, rows - 1) / a.G, hq = h * a.G + min(i, rows - 1) % a.G;
    const int keys = max(0, before + j + 1);
    const int least = max(0, before + min(first + 32 * w, rows - 1) / a.G + 1);  // that all of the wave's rows attend
    const int most = max(0, before + (min(first + ROWS, rows) - 1) / a.G + 1);   // that any of the workgroup's does
    // this workgroup's tiles: one split's share
    const int all_tiles = (most + KT - 1) / KT, split = blockIdx.y, ns = gridDim.y;
    const int t0 = (int)((int64_t)split * all_tiles / ns), nt = (int)((int64_t)(split + 1) * all_tiles / ns);

    // The query: step c of the product contracts over elements 16 c + 8 hh .. + 7.
    h8 q[M::Q][2 * NB];
    float rs = fabsf(a.sl2);
    Eight<DT> qx[2 * NB];
    auto load_q = [&]() __attribute__((always_inline)) {
        const int64_t qi = (int64_t)(start + j) * a.q_stride + (int64_t)hq * D + 8 * hh;
#pragma unroll
        for (int c = 0; c < 2 * NB; c++) qx[c].load(a.q, qi + 16 * c);
    };
    auto make_q = [&]() __attribute__((always_inline)) {
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < 2 * NB; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(qx[c].get(e)));
        float sc = 1.0f;
        if constexpr (DT != TN_F16) {
            sc = row_scale(xor32_max(top));
            rs = rs / sc;
        }
        // a positive factor, so that it can be taken out of the maximum
        rs = fmaxf(rs, 1.1754944e-38f);
        if (a.sl2 < 0.0f) sc = -sc;
#pragma unroll
        for (int c = 0; c < 2 * NB; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = qx[c].get(e) * sc;
                const _Float16 hi = (_Float16)v;
                q[0][c][e] = hi;
                if constexpr (M::Q == 2) q[1][c][e] = (_Float16)(v - (float)hi);
            }
    };
    constexpr int U = KT / 32;
    struct Scores {
        f32x16 s[U];
    };
    struct Probs {
        uint32_t h[KT / 4], l[KT / 4];
    };
    f32x16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[b][e] = 0.0f;
    float m = -INFINITY, l = 0.0f, vref = VREF_MIN;

    // ---- this thread's part of a tile: its loads, and their way into LDS. A wave unpacks of
    // one block of sixteen keys, WPB waves a block, pieces (key, 16 elements) of K and
    // (element) of V
    const int32_t* table = a.table + (int64_t)r * a.width;
    const int blk = w / WPB, id0 = w % WPB * 64 + lane;
    auto on = [&](int x) { return 32 * NB % (64 * WPB) == 0 || id0 + 64 * WPB * x < 32 * NB; };
    struct Pieces {
        uint32_t c[N][4];
    } kr, vr;
    // (tiles past the last are the last again)
    auto page_of = [&](int t) __attribute__((always_inline)) {
        return scalar(table + min((KT * min(t, nt - 1) + 16 * blk) >> a.c.shift, a.width - 1));
    };
    // the plane row of the first of the wave's sixteen keys
    auto row_of = [&](int page, int t) __attribute__((always_inline)) {
        const bool bad = (unsigned)page >= (unsigned)a.c.pages;  // its scales are written so that it does not count
        return (((int64_t)(bad ? 0 : page) * a.c.H + h) << a.c.shift) + ((KT * min(t, nt - 1) + 16 * blk) & (S - 1));
    };
    auto load_k = [&](Pieces& y, int page, int t) __attribute__((always_inline)) {
        const uint8_t* p = a.c.kc + row_of(page, t) * D;
#pragma unroll
        for (int x = 0; x < N; x++) {
            const int id = on(x) ? id0 + 64 * WPB * x : 0;
            load_words(p + (uint32_t)((id & 15) * D + (id >> 4) * 16), y.c[x]);
        }
    };
    auto load_v = [&](Pieces& y, int page, int t) __attribute__((always_inline)) {
        const uint8_t* p = a.c.vc + row_of(page, t) * D;
#pragma unroll
        for (int x = 0; x < N; x++) load_words(p + (uint32_t)((on(x) ? id0 + 64 * WPB * x : 0) * 16), y.c[x]);
    };
    auto unpack_k = [&](int x, int half, int t) __attribute__((always_inline)) {  // eight codes
        const int id = id0 + 64 * WPB * x;
        if (on(x))
            *reinterpret_cast<h8*>(lds + (t & 1) * M::STAGE + (16 * blk + (id & 15)) * M::KP + (id >> 4) * 32 + half * 16) =
                codes8(kr.c[x][2 * half], kr.c[x][2 * half + 1]);
    };
    auto unpack_v = [&](int x, int half, int t) __attribute__((always_inline)) {  // tokens 4 half .. + 3 and 8 + 4 half .. + 3
        const int id = id0 + 64 * WPB * x;
        if (on(x))
            *reinterpret_cast<h8*>(lds + (t & 1) * M::STAGE + M::KB + id * M::VP + (2 * blk + half) * 16) =
                codes8(vr.c[x][half], vr.c[x][2 + half]);
    };
    // The scales, by the first BL lanes of the last wave, a block each.
    const bool scaler = w == 3;
    float ref = VREF_MIN, sk = 0.0f, sv = 0.0f;
    int spage = 0;
    auto scale_page = [&](int t) __attribute__((always_inline)) {
        spage = table[min((KT * min(t, nt - 1) + 16 * (lane & (BL - 1))) >> a.c.shift, a.width - 1)];
    };
    auto load_scales = [&](int t) __attribute__((always_inline)) {
        const bool bad = (unsigned)spage >= (unsigned)a.c.pages;
        const int at = KT * min(t, nt - 1) + 16 * (lane & (BL - 1));
        const int64_t row = ((((int64_t)(bad ? 0 : spage) * a.c.H + h) << a.c.shift) + (at & (S - 1))) >> 4;
        const float k = a.c.ks[row], v = a.c.vs[row];
        sk = bad ? NAN : k;                       // its scores, and so the rows that attend it, are NaN
        sv = bad || at >= len ? 0.0f : v;         // blocks that no row attends count as zeros
    };
    auto write_scales = [&](int t) __attribute__((always_inline)) {
        const float top = quad_max<BL>(sv), next = top >= ref ? vref_for(top) : ref, inv = vref_inverse(next);
        const float share = sv * inv;
        const int small = __any(share < LEAST_SHARE);
        Scales& sc = scales[t & 3];
        if (lane < BL) {
            sc.ks[lane] = sk;
            sc.vs[lane] = sv;
            sc.log[lane] = __builtin_amdgcn_logf(share);
            sc.inv[lane] = __builtin_amdgcn_rcpf(share);
            if (lane == 0) sc.step = ref * inv, sc.vref = next, sc.small = small;
        }
        ref = next;
    };

    // ---- products, in groups of four fragments out of LDS, each group read while the one
    // before it is multiplied: PG of O^T += V^T P^T (a group is 16 keys and up to four blocks
    // of elements), then SG of S^T (XG steps of all the tile's keys).
    constexpr int BG = 4, PB = (NB + BG - 1) / BG, PG = KT / 16 * PB;
    constexpr int XG = 4 / U, SG = (2 * NB + XG - 1) / XG, G = PG + SG;
    h8 f[2][4];
    auto fetch = [&](int n, int slot) __attribute__((always_inline)) {
        if (n < PG) {
            const uint8_t* st = lds + slot * M::STAGE + M::KB + col * M::VP + hh * 16 + n / PB * 32;
#pragma unroll
            for (int e = 0; e < BG; e++)
                if (n % PB * BG + e < NB) f[n & 1][e] = *reinterpret_cast<const h8*>(st + 32 * (n % PB * BG + e) * M::VP);
        } else if (n < G) {
            const uint8_t* st = lds + slot * M::STAGE + col * M::KP + hh * 16;
#pragma unroll
            for (int x = 0; x < XG; x++)
#pragma unroll
                for (int u = 0; u < U; u++)
                    if ((n - PG) * XG + x < 2 * NB)
                        f[n & 1][x * U + u] = *reinterpret_cast<const h8*>(st + 32 * u * M::KP + 32 * ((n - PG) * XG + x));
        }
    };
    auto multiply = [&](int n, const Probs& p, Scores& s) __attribute__((always_inline)) {
        if (n < PG) {
            const int k = 4 * (n / PB);
            const h8 p0 = as_h8(p.h[k], p.h[k + 1], p.h[k + 2], p.h[k + 3]);
            const h8 p1 = M::P == 2 ? as_h8(p.l[k], p.l[k + 1], p.l[k + 2], p.l[k + 3]) : p0;
#pragma unroll
            for (int e = 0; e < BG; e++) {
                const int b = n % PB * BG + e;
                if (b >= NB) continue;
                if (M::P == 2) o[b] = El<true>::mfma(f[n & 1][e], p1, o[b]);
                o[b] = El<true>::mfma(f[n & 1][e], p0, o[b]);
            }
        } else {
            if (n == PG) {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s.s[u][e] = 0.0f;
            }
#pragma unroll
            for (int x = 0; x < XG; x++) {
                const int c = (n - PG) * XG + x;
                if (c >= 2 * NB) continue;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (M::Q == 2) s.s[u] = El<true>::mfma(f[n & 1][x * U + u], q[M::Q - 1][c], s.s[u]);
                    s.s[u] = El<true>::mfma(f[n & 1][x * U + u], q[0][c], s.s[u]);
                }
            }
        }
    };

    // 16-bit rows have the blocks' shares in the exponents where they can, f32 rows as a product,
    // which keeps its digits.
    constexpr bool FOLD = DT != TN_F32;
    Scores s;
    Probs p;
    auto turn = [&](auto last_turn, int t) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last_turn)::value;
        constexpr int END = LAST ? PG : G;
        const Scales& sc = scales[t & 3];
        float fs[BL], mb[BL];
#pragma unroll
        for (int b = 0; b < BL; b++) fs[b] = rs * sc.ks[b];
        // the products' wait states: the compiler does not see that max3f's assembly reads their result
        __builtin_amdgcn_sched_barrier(0);
#if __HIP_DEVICE_COMPILE__
        asm volatile("s_nop 15\n\ts_nop 1");
#endif
        __builtin_amdgcn_sched_barrier(0);
        const bool edge = KT * t + KT > least;  // uniform, and so for all tiles behind
        float step = sc.step;
        if (edge) {
            // keys that a row does not attend, and the reference for scales of its own keys alone: what
            // later tokens hold costs a row no digits
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < BL; b++) top = fmaxf(top, KT * t + 16 * b < keys ? sc.vs[b] : 0.0f);
            const float next = top >= vref ? vref_for(top) : vref;
            step = vref * vref_inverse(next);
            vref = next;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int k = KT * t + 32 * u + 8 * (e >> 2) + 4 * hh + (e & 3);
                    const float v = s.s[u][e] * fs[2 * u + (e >> 3)];
                    s.s[u][e] = k >= keys ? -INFINITY : v;
                }
#pragma unroll
            for (int b = 0; b < BL; b++) fs[b] = 1.0f;
        } else {
            vref = sc.vref;
        }
#pragma unroll
        for (int b = 0; b < BL; b++) {
            const f32x16& x = s.s[b >> 1];
            const int e = 8 * (b & 1);
            mb[b] = max3f(max3f(x[e], x[e + 1], x[e + 2]), max3f(x[e + 3], x[e + 4], x[e + 5]),
                          max3f(x[e + 6], x[e + 7], x[e + 7])) * fs[b];
        }
        const float mx = xor32_max(max3f(mb[0], mb[1], BL == 4 ? fmaxf(mb[BL - 2], mb[BL - 1]) : mb[1]));
        const bool grew = __any(mx > m + RESCALE_SLACK);
        if (grew || __any(step != 1.0f)) {
            float al = step;
            if (grew) {
                const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= f;
                al *= f;
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[b][e] *= al;
        }
        const float mu = P_BIAS - (m == -INFINITY ? 0.0f : m);
        auto probabilities = [&](auto fold, int b) __attribute__((always_inline)) {  // of a block
            constexpr bool IN = decltype(fold)::value;  // its share is in the exponent
            const float ma = IN ? mu + sc.log[b] : mu;
            // (of a block that the row does not attend it may be anything: held to 1)
            const float share = IN ? 1.0f : fminf(sc.vs[b] * vref_inverse(vref), 1.0f);
            float lb = 0.0f;
#pragma unroll
            for (int e = 8 * (b & 1); e < 8 * (b & 1) + 8; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s.s[b >> 1][e], fs[b], ma));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s.s[b >> 1][e + 1], fs[b], ma));
                const int x = 8 * (b >> 1) + e / 2;
                if constexpr (IN) {
                    split_p<M::P>(p0, p1, p.h[x], p.l[x], lb);
                } else {
                    float none = 0.0f;
                    lb += p0;
                    lb += p1;
                    split_p<M::P>(p0 * share, p1 * share, p.h[x], p.l[x], none);
                }
            }
            l = IN ? fmaf(lb, sc.inv[b], l) : l + lb;
        };
        if (FOLD && !edge && !__builtin_amdgcn_readfirstlane(sc.small)) {
#pragma unroll
            for (int b = 0; b < BL; b++) probabilities(std::integral_constant<bool, FOLD>{}, b);
        } else {
#pragma unroll
            for (int b = 0; b < BL; b++) probabilities(std::false_type{}, b);
        }
        // computed here, not where the products take them
#if __HIP_DEVICE_COMPILE__
#pragma unroll
        for (int e = 0; e < KT / 4; e++) {
            asm volatile("" : "+v"(p.h[e]));
            if constexpr (M::P == 2) asm volatile("" : "+v"(p.l[e]));
        }
        asm volatile("" : "+v"(l));
#endif
        const int vslot = t & 1;
        fetch(0, vslot);
        __builtin_amdgcn_s_setprio(1);  // the products' few instructions ahead of the other wave's many
        // eight codes of V or of K at a time, then the next loads
        constexpr int WORK = LAST ? 0 : 4 * N + 1;
        auto work = [&](int x) __attribute__((always_inline)) {
            if (x < 2 * N) unpack_v(x >> 1, x & 1, t + 1);
            else if (x < 4 * N) unpack_k(x / 2 - N, x & 1, t + 2);
            else {
                load_v(vr, page_of(t + 2), t + 2);
                load_k(kr, page_of(t + 3), t + 3);
            }
        };
#pragma unroll
        for (int n = 0; n < END; n++) {
            __builtin_amdgcn_sched_barrier(0);
            if (n + 1 < END) fetch(n + 1, n + 1 < PG ? vslot : vslot ^ 1);
            multiply(n, p, s);
#pragma unroll
            for (int x = n * WORK / G; x < (n + 1) * WORK / G; x++) work(x);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!LAST) {
            if (scaler) {
                write_scales(t + 2);
                load_scales(t + 3);
                scale_page(t + 4);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (!LAST) __syncthreads();
    };
    if (nt > t0) {
        // all that the first tiles need is asked for before any of it is waited for
        Pieces k1;
        load_q();
        load_k(k1, page_of(t0), t0), load_k(kr, page_of(t0 + 1), t0 + 1);
        load_v(vr, page_of(t0), t0);
        if (scaler) {
            for (int t = t0; t < t0 + 2; t++) scale_page(t), load_scales(t), write_scales(t);
            scale_page(t0 + 2);
            load_scales(t0 + 2);
            scale_page(t0 + 3);
        }
        make_q();
        const Pieces k2 = kr;
        kr = k1;
#pragma unroll
        for (int x = 0; x < 2 * N; x++) unpack_k(x >> 1, x & 1, t0);
        kr = k2;
#pragma unroll
        for (int x = 0; x < 2 * N; x++) unpack_k(x >> 1, x & 1, t0 + 1);
        load_k(kr, page_of(t0 + 2), t0 + 2);
#pragma unroll
        for (int x = 0; x < 2 * N; x++) unpack_v(x >> 1, x & 1, t0);
        load_v(vr, page_of(t0 + 1), t0 + 1);
        __syncthreads();
        fetch(PG, t0 & 1);
#pragma unroll
        for (int n = PG; n < G; n++) {
            if (n + 1 < G) fetch(n + 1, t0 & 1);
            multiply(n, p, s);
        }
        __syncthreads();
        for (int t = t0; t + 1 < nt; t++) turn(std::false_type{}, t);
        turn(std::true_type{}, nt - 1);
    }

    // the last products' wait states, whatever their first reader is
    __builtin_amdgcn_sched_barrier(0);
#if __HIP_DEVICE_COMPILE__
    asm volatile("s_nop 15\n\ts_nop 1");
#endif
    __builtin_amdgcn_sched_barrier(0);
    // out through LDS, so that a row's bytes leave together, in `type` to rows of a.out or (many_o) f32
    l = xor32_sum(l);
    uint8_t* mine = lds + w * 32 * M::OP;
    __syncthreads();
    auto leave = [&](auto type, float f, float g) __attribute__((always_inline)) {
        constexpr int OT = type.value, SIZE = OT == TN_F32 ? 4 : 2;
#pragma unroll
        for (int b0 = 0; b0 < NB; b0 += 4) {  // four blocks at a time
            const int nb = NB - b0 < 4 ? NB - b0 : 4, pieces = nb * 2 * SIZE;  // of 16 bytes, a row
#pragma unroll
            for (int b = b0; b < b0 + nb; b++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float y[4] = {o[b][e] * f * g, o[b][e + 1] * f * g, o[b][e + 2] * f * g, o[b][e + 3] * f * g};
                    uint8_t* p = mine + col * M::OP + (32 * (b - b0) + 2 * e + 4 * hh) * SIZE;
                    if constexpr (OT == TN_F32) {
                        *reinterpret_cast<f32x4*>(p) = (f32x4){y[0], y[1], y[2], y[3]};
                    } else {
                        using E = El<OT == TN_F16>;
                        *reinterpret_cast<uint2*>(p) = make_uint2(E::pack_out(y[0], y[1]), E::pack_out(y[2], y[3]));
                    }
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own rows
#pragma unroll
            for (int k = 0; k < pieces / 2; k++) {
                const int x = lane + 64 * k, rr = x / pieces, ii = first + 32 * w + rr;
                typedef uint32_t u4 __attribute__((ext_vector_type(4)));
                typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
                const u4 v = *reinterpret_cast<const u4*>(mine + rr * M::OP + x % pieces * 16);
                int64_t row = (int64_t)(start + ii / a.G) * a.Hq + h * a.G + ii % a.G;
                if (ns > 1) row = row * ns + split;
                char* to = ns > 1 ? reinterpret_cast<char*>(a.many_o) : static_cast<char*>(a.out);
                if (ii < rows) *reinterpret_cast<v4*>(to + (row * D + 32 * b0) * SIZE + x % pieces * 16) = v;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    };
    const int64_t row = (int64_t)(start + j) * a.Hq + hq;
    if (ns > 1) {  // a split's part: k_paged8_join's
        leave(std::integral_constant<int, TN_F32>{}, 1.0f, 1.0f);
        if (hh == 0 && i < rows) reinterpret_cast<Part*>(a.many_ml)[row * ns + split] = Part{m, l, vref, 0.0f};
    } else {
        leave(std::integral_constant<int, DT>{}, 1.0f / l, vref);
        if (a.lse && hh == 0 && i < rows) a.lse[row] = l == 0.0f ? -INFINITY : (m - P_BIAS) * LN2 + logf(l);
    }
}

template <int DT, int NB>
__global__ __launch_bounds__(256, (Many8<DT, NB>::WAVES)) void k_paged8_many(const Paged8Args a, int tiles) {
    constexpr int ROWS = MANY_ROWS;
    __shared__ __align__(16) uint8_t lds[Many8<DT, NB>::LDS_BYTES];
    __shared__ __align__(16) Scales scales[4];
    // the longest rows first; a key/value head's workgroups on the same die when there are eight
    const int h = (int)blockIdx.x % a.c.H, tile = tiles - 1 - (int)blockIdx.x / a.c.H;
    int r = 0;
    {  // request r has tiles row_start[r] G / ROWS + r and on: at least as many as its rows need
        int hi = a.n;
        while (hi - r > 1) {
            const int mid = (r + hi) >> 1;
            if ((int)((int64_t)start_of(a, mid) * a.G / ROWS) + mid <= tile) r = mid;
            else hi = mid;
        }
    }
    const int start = start_of(a, r), all = rows_of(a, r, start);
    const int first = (tile - (int)((int64_t)start * a.G / ROWS) - r) * ROWS;
    const int rows = min(all, a.max_rows) * a.G;
    if (first < 0 || first >= rows || rows <= a.few) return;  // few rows: k_paged8_few's
    const int len = max(0, min(a.lens[r], a.max_len)), before = len - all;
    many8_tile<DT, NB>(a, lds, scales, h, r, start, rows, first, len, before);
}

// The splits of k_paged8_many's rows, in order: four output columns a thread.
template <int DT>
__global__ __launch_bounds__(256) void k_paged8_join(const Paged8Args a, int ns) {
    const int D = 32 * a.c.nb, q4 = D / 4;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = e / q4;
    const int d = (int)(e - row * q4) * 4, t = (int)(row / a.Hq);
    if (t >= start_of(a, a.n)) return;
    int r = 0, hi = a.n;  // the row's request
    while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (start_of(a, mid) <= t) r = mid;
        else hi = mid;
    }
    const int start = start_of(a, r), c = min(rows_of(a, r, start), a.max_rows);
    if (t < start || t - start >= c || c * a.G <= a.few) return;  // (rows ahead of the first request's are no one's)
    join<DT>(a, a.many_o + row * ns * D + d, reinterpret_cast<const Part*>(a.many_ml) + row * ns, ns, d, [&]() { return row; });
}

// Splits of the keys of k_paged8_few: one round of the workgroups that compute units
// hold, of 512 keys or more, up to eight of them of 256. Against a round of 1024 workgroups,
// us: sixteen bf16 tokens over 512 to 4096 keys, 32/8 heads of 128 elements, 22.3 / 24.5, of 256
// elements 48.7 / 55.5; sixty-four over 1000 to 3000 56 / 62; one over 8000 13.5 / 13.4.
constexpr int64_t FEW_WGS = 512, FEW_KEYS = 512, FEW_MAX_SPLIT = 64;
int64_t few_most(int64_t max_len) {
    if (max_len <= FEW_KEYS) return 1;
    return std::max(std::min<int64_t>(cdiv(max_len, 256), 8), std::min(cdiv(max_len, FEW_KEYS), FEW_MAX_SPLIT));
}
int few_splits(const Pages8& c, int64_t n, int64_t few, int64_t max_len) {
    const int64_t wgs = std::max<int64_t>(1, n * c.H * cdiv(few, 16));
    return (int)std::max<int64_t>(1, std::min(FEW_WGS / wgs, few_most(max_len)));
}

tn_status attn_check(const char* op, const tn_q8_cache* cache, int64_t n, int64_t tokens, int64_t Hq, int64_t max_rows,
                     int64_t max_len, Pages8* c) {
    TN_TRY(paged_check(op, cache, c));
    if (n < 0 || tokens < 0 || Hq < 0 || max_rows < 0 || max_len < 0)
        return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    if (Hq % c->H)
        return fail(TN_ENOTIMPL, std::string(op) + ": " + std::to_string(Hq) + " query heads do not divide into " +
                                     std::to_string(c->H) + " key/value heads");
    if (n > 65535 || Hq > 65535 || tokens > INT32_MAX || tokens * Hq > (1 << 30) || n * c->H > (1 << 21) ||
        max_len > (1 << 30))
        return fail(TN_EVALUE, std::string(op) + ": shape too large");
    return TN_OK;
}

// Rows of its partials at most, for this call and every smaller one: no more than
// FEW_WGS workgroups of 16 rows, splits counted.
int64_t part_rows(const Pages8& c, int64_t n, int64_t few, int64_t max_len) {
    const int64_t most = few_most(max_len);
    return most < 2 ? 0 : std::min(std::min<int64_t>(few, 16) * FEW_WGS, n * c.H * few * most);
}

// Splits of the keys of k_paged8_many: what fills one round of the workgroups that compute units
// hold, two each, of 512 keys or more of a request's middle row. us at rounds of 256 / 512 / 1024
// workgroups, bf16, 32/8 heads of 128 elements: 512 rows behind 20000 tokens 297 / 205 / 224,
// behind 4096 75 / 59 / 72; a prompt of 1024, whose middle row has 512 keys, without splits 37,
// in two 42.
constexpr int64_t MANY_WGS = 512, MANY_MAX_SPLIT = 8;
int many_splits(const Pages8& c, int64_t n, int64_t tokens, int64_t G, int64_t max_rows, int64_t max_len) {
    const int64_t wgs = (tokens * G / MANY_ROWS + n) * c.H, keys = max_len - std::min(max_rows, max_len) / 2;
    return (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(MANY_WGS, wgs), cdiv(keys, 512), MANY_MAX_SPLIT}));
}
// Rows of its partials at most, for this call and every smaller one: above one split there
// are under MANY_WGS workgroups a split.
int64_t many_rows(const Pages8& c, int64_t tokens, int64_t G, int64_t max_len) {
    const int64_t most = std::min(cdiv(max_len, 512), MANY_MAX_SPLIT);
    return most < 2 ? 0 : std::min(tokens * G * c.H * most, 2 * MANY_WGS * MANY_ROWS);
}

// Which kernel takes a request's rows. k_paged8_few reads and unpacks the codes again for
// every 16 folded rows but starts at once and splits finely; k_paged8_many fills 128
// rows, and its tiles follow one another. So k_paged8_few takes all rows of a call whose
// products (tokens * Hq * max_len * D) are few, and of a larger call the requests of up to
// FEW_ROWS folded rows, if it is of several. How many are few: a tile of k_paged8_many has
// the same softmax and the same barriers for rows of 64 elements as for 128, so those wait
// longer for it. Few against many, us, bf16: 64 elements, products / 2^30: 2 33 / 40, 4 48 / 50,
// 8 62 / 55, 9 62 / 66 (six ragged requests 6 45 / 58); 128: 2 31 / 32 and 33 / 36, 4 50 / 43 (ragged: 8
// 64 / 65, 12 88 / 79); 256: 8 97 / 94, 16 157 / 111. f32, 128: 2 32 / 38, 4 56 / 54, 8 97 / 82. Its grid
// is as long for every request as for the longest: up to FEW_GRID workgroups of it.
constexpr int FEW_ROWS = 128;
constexpr int64_t FEW_GRID = 8192;
int64_t few_products(int nb) { return nb <= 3 ? 7ll << 30 : 3ll << 30; }

// Folded rows of a request that k_paged8_few takes at most in this call; 0: it is not launched.
int64_t few_limit(const Pages8& c, int64_t n, int64_t tokens, int64_t G, int64_t max_rows, int64_t max_len) {
    const int64_t rows = max_rows * G;
    // (tokens * Hq is at most 2^30, D 2^8)
    const bool little = tokens * G * c.H * 32 * c.nb <= few_products(c.nb) / std::max<int64_t>(max_len, 1) &&
                        n * c.H * cdiv(rows, 16) <= FEW_GRID;
    return rows <= FEW_ROWS || little ? rows : n > 1 ? FEW_ROWS : 0;
}

int64_t work_rows(const Pages8& c, int64_t n, int64_t tokens, int64_t G, int64_t max_rows, int64_t max_len) {
    return part_rows(c, n, max_rows * G, max_len) + (max_rows * G > FEW_ROWS ? many_rows(c, tokens, G, max_len) : 0);
}

template <int DT, int NB>
tn_status launch_at(hipStream_t st, const Paged8Args& a, int64_t tokens) {
    if (a.few) {
        const dim3 grid((unsigned)a.nsplit, (unsigned)(a.c.H * cdiv(a.few, 16)), (unsigned)a.n);
        hipLaunchKernelGGL((k_paged8_few<DT, NB>), grid, dim3(256), 0, st, a);
        TN_LAUNCHED();
    }
    if ((int64_t)a.max_rows * a.G > a.few) {
        const int ns = many_splits(a.c, a.n, tokens, a.G, a.max_rows, a.max_len);
        const int64_t tiles = tokens * a.G / MANY_ROWS + a.n;
        const dim3 grid((unsigned)(tiles * a.c.H), (unsigned)ns);
        hipLaunchKernelGGL((k_paged8_many<DT, NB>), grid, dim3(256), 0, st, a, (int)tiles);
        TN_LAUNCHED();
        if (ns > 1) {
            const int64_t quads = tokens * a.Hq * (8 * NB);
            hipLaunchKernelGGL(k_paged8_join<DT>, dim3((unsigned)cdiv(quads, 256)), dim3(256), 0, st, a, ns);
            TN_LAUNCHED();
        }
    }
    if (a.few && a.nsplit > 1) {
        const dim3 grid((unsigned)cdiv((int64_t)a.few * (8 * NB), 64), (unsigned)a.c.H, (unsigned)a.n);
        hipLaunchKernelGGL(k_paged8_combine<DT>, grid, dim3(64), 0, st, a);
        TN_LAUNCHED();
    }
    return TN_OK;
}

template <int DT>
tn_status launch(hipStream_t st, const Paged8Args& a, int64_t tokens) {
    switch (a.c.nb) {
        case 1: return launch_at<DT, 1>(st, a, tokens);
        case 2: return launch_at<DT, 2>(st, a, tokens);
        case 3: return launch_at<DT, 3>(st, a, tokens);
        case 4: return launch_at<DT, 4>(st, a, tokens);
        case 5: return launch_at<DT, 5>(st, a, tokens);
        case 6: return launch_at<DT, 6>(st, a, tokens);
        case 7: return launch_at<DT, 7>(st, a, tokens);
        default: return launch_at<DT, 8>(st, a, tokens);
    }
}

}  // namespace
}  // namespace tn

using namespace tn;

extern "C" {

int64_t tn_sdpa_paged_q8_work_floats(const tn_q8_cache* cache, int64_t n, int64_t tokens, int64_t Hq, int64_t max_rows,
                                     int64_t max_len) {
    Pages8 c;
    if (attn_check("sdpa_paged_q8_work_floats", cache, n, tokens, Hq, max_rows, max_len, &c) != TN_OK) return 0;
    if (!n || !tokens || !Hq || !max_rows) return 0;
    return work_rows(c, n, tokens, Hq / c.H, std::min(max_rows, tokens), max_len) * (32 * c.nb + 4);
}

tn_status tn_sdpa_paged_q8(void* stream, const tn_q8_cache* cache, int dtype, const void* q, int64_t q_stride,
                           int64_t tokens, int64_t Hq, int64_t n, const int32_t* row_start, const int32_t* lens,
                           const int32_t* table, int64_t width, int64_t max_rows, int64_t max_len, double scale,
                           float* work, int64_t work_floats, void* out, float* lse) {
    const char* op = "sdpa_paged_q8";
    Paged8Args a{};
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, "sdpa_paged_q8: rows must be float32, bfloat16 or float16");
    TN_TRY(attn_check(op, cache, n, tokens, Hq, max_rows, max_len, &a.c));
    const int64_t D = 32 * a.c.nb, G = Hq / a.c.H;
    if (width < 0 || width > INT32_MAX || max_len > (width << a.c.shift))
        return fail(TN_EINVAL, "sdpa_paged_q8: max_len " + std::to_string(max_len) + " is past what " +
                                   std::to_string(width) + " pages hold");
    if (tokens > 1 && q_stride < Hq * D) return fail(TN_EINVAL, "sdpa_paged_q8: the row stride is shorter than a row");
    if (tokens > 1 && q_stride > INT64_MAX / 8 / tokens) return fail(TN_EVALUE, "sdpa_paged_q8: shape too large");
    if (max_len && !a.c.pages) return fail(TN_EINVAL, "sdpa_paged_q8: the cache has no pages");
    const int64_t need = tn_sdpa_paged_q8_work_floats(cache, n, tokens, Hq, max_rows, max_len);
    if (work_floats < need)
        return fail(TN_EVALUE, "sdpa_paged_q8: work holds " + std::to_string(work_floats) +
                                   " floats, this call needs " + std::to_string(need));
    if (!n || !tokens || !Hq || !max_rows) return TN_OK;
    if (!q || !out || !row_start || !lens || (max_len && !table) || (need && !work))
        return fail(TN_EVALUE, "sdpa_paged_q8: null pointer");
    if (reinterpret_cast<uintptr_t>(work) & 15) return fail(TN_EVALUE, "sdpa_paged_q8: work must be 16-byte aligned");
    TN_TRY(paged_check_planes(op, a.c));
    const double sc = std::isnan(scale) ? 1.0 / std::sqrt((double)D) : scale;
    a.q = q, a.out = out, a.lse = lse, a.row_start = row_start, a.lens = lens, a.table = table;
    a.q_stride = q_stride, a.n = (int)n, a.tokens = (int)tokens, a.Hq = (int)Hq, a.G = (int)G, a.width = (int)width;
    a.max_rows = (int)std::min(max_rows, tokens), a.max_len = (int)max_len;
    a.sl2 = (float)(sc * 1.4426950408889634);
    a.few = (int)few_limit(a.c, n, tokens, G, a.max_rows, max_len);
    a.nsplit = few_splits(a.c, n, a.few, max_len);
    // f32 rows, then their parts: the few's and the many's
    const int64_t few = part_rows(a.c, n, a.max_rows * G, max_len);
    const int64_t rows = work_rows(a.c, n, tokens, G, a.max_rows, max_len);
    a.part_o = work, a.many_o = work + few * D;
    a.part_ml = reinterpret_cast<float2*>(work + rows * D), a.many_ml = a.part_ml + 2 * few;  // (Part: two each)
    hipStream_t st = (hipStream_t)stream;
    const Turn turn(stream);
    if (dtype == TN_F32) return launch<TN_F32>(st, a, tokens);
    if (dtype == TN_BF16) return launch<TN_BF16>(st, a, tokens);
    return launch<TN_F16>(st, a, tokens);
}

}  // extern "C"
