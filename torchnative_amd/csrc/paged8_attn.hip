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

// k_paged8_few's parts of each 16-bit operand: a 16-bit query is one f16 (a bf16 row
// scaled by a power of two), an f32 one two; probabilities are two for an output of 11
// or 24 bits, one for 8.
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

// The scale of values that a wave's sums are held under: a power of two above every block's
// scale met so far, so that a probability times its block's share of it is at most itself.
TN_INLINE float vref_for(float scale) {
    const uint32_t e = (__builtin_bit_cast(uint32_t, scale) >> 23) & 0xffu;
    return __builtin_bit_cast(float, min(e + 1u, 253u) << 23);
}
constexpr float VREF_MIN = 1.1754943508222875e-38f;  // 2^-126

// ---- few rows ---------------------------------------------------------------------
//
// A wave takes 64 keys at a time, four blocks. Tile t (0 .. 3) of S^T has keys
// 16 g + 4 t + i in row 4 g + i (lane c + 16 g holds rows 4 g .. 4 g + 3 of column c),
// so that a lane holds the sixteen keys of one block, whose scales are one number each
// for keys and for values, and the operands of its part of two 32-key products
// O^T += V^T P^T, whose values it reads as sixteen bytes a column.
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
            // values of a block that no row attends count as zeros, whatever its page holds
            if (k0 >= len || x.bad) x.vs = 0.0f;
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
            const float nv = vref_for(mv), al = vref / nv;
            vref = nv;
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) o[b] = o[b] * al;
        }
        const float mu = P_BIAS - (m == -INFINITY ? 0.0f : m), share = x.vs / vref;
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

// Splits of a row, in order (the same bits every time), into four output columns.
template <int DT>
TN_INLINE void join(const Paged8Args& a, const float* po, const Part* ml, int ns, int64_t row, int d) {
    const int D = 32 * a.c.nb;
    float mm = -INFINITY, tl = 0.0f, vv = 0.0f;
    for (int s = 0; s < ns; s++) mm = fmaxf(mm, ml[s].m), vv = fmaxf(vv, ml[s].v);
    const float mu = mm == -INFINITY ? 0.0f : mm;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < ns; s++) {
        const Part p = ml[s];
        const float f = exp2f(p.m - mu), fv = f * (p.v / vv);
        tl += p.l * f;
        const f32x4 v = *reinterpret_cast<const f32x4*>(po + (int64_t)s * D);
#pragma unroll
        for (int n = 0; n < 4; n++) acc[n] += v[n] * fv;
    }
    const float inv = 1.0f / tl;
    const float y[4] = {acc[0] * inv * vv, acc[1] * inv * vv, acc[2] * inv * vv, acc[3] * inv * vv};
    store4<DT>(a.out, row * D + d, y);
    if (a.lse && d == 0) a.lse[row] = tl == 0.0f ? -INFINITY : (mm - P_BIAS) * LN2 + logf(tl);
}

template <int DT>
__global__ __launch_bounds__(256) void k_paged8_combine(const Paged8Args a) {
    const int D = 32 * a.c.nb, q4 = D / 4;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t pr = e / q4;
    const int d = (int)(e - pr * q4) * 4;
    const int i = (int)(pr % a.few);
    const int64_t rh = pr / a.few;
    const int h = (int)(rh % a.c.H);
    const int64_t r = rh / a.c.H;
    if (r >= a.n) return;
    const int start = start_of(a, r), c = min(rows_of(a, r, start), a.max_rows);
    if (i >= c * a.G || c * a.G > a.few) return;
    const int64_t row = (int64_t)(start + i / a.G) * a.Hq + h * a.G + i % a.G;
    join<DT>(a, a.part_o + pr * a.nsplit * D + d, reinterpret_cast<const Part*>(a.part_ml) + pr * a.nsplit, a.nsplit, row,
             d);
}

// Splits of the keys of k_paged8_few: one round of the workgroups that compute units
// hold, of 512 keys or more, up to eight of them of 256.
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

int64_t work_rows(const Pages8& c, int64_t n, int64_t tokens, int64_t G, int64_t max_rows, int64_t max_len) {
    (void)tokens;
    return part_rows(c, n, max_rows * G, max_len);
}

template <int DT, int NB>
tn_status launch_at(hipStream_t st, const Paged8Args& a, int64_t tokens) {
    (void)tokens;
    if (a.few) {
        const dim3 grid((unsigned)a.nsplit, (unsigned)(a.c.H * cdiv(a.few, 16)), (unsigned)a.n);
        hipLaunchKernelGGL((k_paged8_few<DT, NB>), grid, dim3(256), 0, st, a);
        TN_LAUNCHED();
    }
    if (a.few && a.nsplit > 1) {
        const int64_t rows = (int64_t)a.n * a.c.H * a.few;
        hipLaunchKernelGGL(k_paged8_combine<DT>, dim3((unsigned)cdiv(rows * (8 * NB), 256)), dim3(256), 0, st, a);
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
    a.few = (int)(a.max_rows * G);
    a.nsplit = few_splits(a.c, n, a.few, max_len);
    const int64_t rows = work_rows(a.c, n, tokens, G, a.max_rows, max_len);
    a.part_o = work;
    a.part_ml = reinterpret_cast<float2*>(work + rows * D);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) return launch<TN_F32>(st, a, tokens);
    if (dtype == TN_BF16) return launch<TN_BF16>(st, a, tokens);
    return launch<TN_F16>(st, a, tokens);
}

}  // extern "C"
