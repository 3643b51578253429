// Attention of ragged rows over the paged 4-bit cache (tnhip.h describes the
// planes and the rows).
//
// Rows of a request are folded over the query heads that share a key/value head:
// row i of (request, key/value head) is token i / G, head h * G + i % G, so that
// G heads read each key once. Scores are computed transposed, S^T = K Q^T, and so
// is the output, O^T = V^T P^T: the lane that holds a column's scores then holds
// them as P^T's operand, with no exchange between lanes (below).
#include "paged.h"

#include <algorithm>
#include <cmath>

#include "attn_common.h"

namespace tn {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

struct PagedArgs {
    Pages c;
    const void* q;
    void* out;
    float* lse;  // nullable
    const int32_t *row_start, *lens, *table;
    int64_t q_stride;
    int n, tokens, Hq, G, width, max_rows, max_len;  // G = Hq / H
    float sl2;        // scale * log2(e)
    int nsplit;       // k_paged_few: splits of the keys
    int few;          // requests of more folded rows are k_paged_many's; 0: all are
    float* part_o;    // [n][H][few][nsplit][D] and
    float2* part_ml;  // [n][H][few][nsplit], above one split
    float* many_o;    // k_paged_many's: [tokens][Hq][splits][D] and
    float2* many_ml;  // [tokens][Hq][splits], above one split
};

// Probabilities are kept at 2^P_BIAS times their size over the running maximum,
// which may lag by RESCALE_SLACK: at most 2^14, so that f16 holds them, and those
// far below the maximum stay out of its subnormal range as long as they count.
constexpr float P_BIAS = 6.0f;

// k_paged_few's parts of each 16-bit operand: a 16-bit query is one f16 (a bf16 row
// scaled by a power of two), an f32 one two; probabilities are two for an output of 11
// or 24 bits, one for 8; values (code * scale, 15 bits) two for 24. One part is a rounding
// of 2^-12 at the mean, which a bf16 output, 2^-9, does not show (off the exact result by
// 1.7e-3 of its norm, as f32 throughout is) and an f16 one shows by a quarter (2.6e-4,
// 2.1e-4 with values in two parts as well). Two parts of both cost bf16 rows 8 % (sixteen
// of 512 to 4096 keys, 18.2 and 19.9 us), of values f16 rows 11 % (twelve of 20000 to
// 40000, 100 and 111).
template <int DT>
struct Parts {
    static constexpr int Q = DT == TN_F32 ? 2 : 1, P = DT == TN_BF16 ? 1 : 2, V = DT == TN_F32 ? 2 : 1;
};

#define TN_INLINE __device__ __attribute__((always_inline)) inline

// row_start[i], and request r's first row and number of rows: within the call's rows,
// whatever row_start holds.
TN_INLINE int start_of(const PagedArgs& a, int i) { return min(max(a.row_start[i], 0), a.tokens); }
TN_INLINE int rows_of(const PagedArgs& a, int r, int start) { return max(start_of(a, r + 1) - start, 0); }

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

// Eight codes of a dword as f16, exactly: its low nibbles (bytes 0 2, bytes 1 3) under
// the bits of 1024, its high ones as 16 times their value there. One v_and_or_b32 a
// pair: an instruction takes one constant, so the bits of 1024 sit in a vector
// register, where the compiler does not see what they are.
struct Unpack {
    uint32_t one, sixty_four;
    TN_INLINE Unpack() {
#if __HIP_DEVICE_COMPILE__
        asm("v_mov_b32 %0, 0x64006400" : "=v"(one));
        asm("v_mov_b32 %0, 0x54005400" : "=v"(sixty_four));
#endif
    }
    TN_INLINE h2 bits(uint32_t w, uint32_t mask) const { return as_h2((w & mask) | one); }
    // 64 more than the nibbles (72 more than the codes), for a product whose sum starts
    // from -72 times the other operand's
    TN_INLINE h8 biased(uint32_t w) const {
        auto bits64 = [&](uint32_t x) { return (x & 0x00F000F0u) | sixty_four; };
        return as_h8(bits64(w << 4), bits64(w >> 4), bits64(w), bits64(w >> 8));
    }
    TN_INLINE void low(uint32_t w, uint32_t& a, uint32_t& b) const {
        const h2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
        a = __builtin_bit_cast(uint32_t, bits(w, 0x000F000Fu) + off);
        b = __builtin_bit_cast(uint32_t, bits(w >> 8, 0x000F000Fu) + off);
    }
    TN_INLINE void high(uint32_t w, uint32_t& a, uint32_t& b) const {
        const h2 r = {(_Float16)0.0625f, (_Float16)0.0625f}, off = {(_Float16)-72.0f, (_Float16)-72.0f};
        a = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(bits(w, 0x00F000F0u), r, off));
        b = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(bits(w >> 8, 0x00F000F0u), r, off));
    }
};

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


// ---- few rows ---------------------------------------------------------------------
//
// A wave takes 32 keys at a time. A 16 x 16 x 32 product contracts over one block of
// 32 elements, so the f32 result is scaled by the block's own scale: codes enter
// the product exactly. Tile t (0, 1) of S^T has keys 8 g + 4 t + i in row 4 g + i
// (lane c + 16 g holds rows 4 g .. 4 g + 3 of column c), so that a lane holds eight
// consecutive keys, the operand of its part of the 32-key product O^T += V^T P^T,
// whose values it reads as two dwords a block and column (tnhip.h: v_codes).
//
// Single rows are bound by the cache's bytes: nothing of a key goes through LDS, a wave
// loads its next tile whole while it computes one, and the splits make one round of the
// resident workgroups. Twelve requests of 20000 to 40000 keys, 8 key/value heads of 128,
// f16: 96 to 100 us with the merge, 4.2 TB/s; 5.2 of requests of one length (else the shorter
// ones' workgroups wait for the longest's). Sixteen of 512 to 4096, bf16: 18 us, 14 and 4 of
// merge, 2.4 TB/s: eight tiles a wave, so that starting and merging count; one of 300, 9
// heads of 64, f32: 5.7 us, a launch and one tile's chain of loads, products, softmax.
// Many rows are bound by the vector unit, which unpacks the codes anew for every 16.
template <int NB>
struct KeyTile {
    uint32_t k[2][NB];    // rows of the two score tiles: this lane's part of each block
    uint32_t kd[4 * NB];  // scales of its part's eight keys, [8][NB] f16
    uint32_t v[2 * NB];   // values of its part's eight keys, a byte column of each block
    uint32_t vd[4 * NB];  // their scales, [NB][8]
    int bad;              // its part's page is outside the cache
};

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

template <int DT, int NB>
__global__ __launch_bounds__(256) void k_paged_few(const PagedArgs a) {
    constexpr int PQ = Parts<DT>::Q, PP = Parts<DT>::P, PV = Parts<DT>::V, D = 32 * NB;
    __shared__ __align__(16) float so[4][16][D + 4];
    __shared__ float2 sml[4][16];
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

    // the query, as f16 parts in the order of the codes' elements
    // (16-bit rows: and what a block's product of codes 72 too large starts from. The f32
    // sums lose four bits by it, 2^-20 of a score, which an f32 row does not spare)
    constexpr bool BIASED = DT != TN_F32 && NB <= 4;  // (more blocks: no registers for it)
    h8 q[PQ][NB];
    f32x4 zero[NB];
    float rs = fabsf(a.sl2);
    {
        float x[NB][8], top = 0.0f;
        const int64_t qi = (int64_t)(start + j) * a.q_stride + (int64_t)hq * D;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float lo[4], hi[4];
            load4<DT>(a.q, qi + 32 * b + 4 * g, lo);
            load4<DT>(a.q, qi + 32 * b + 16 + 4 * g, hi);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[b][e] = lo[((e & 1) << 1) | (e >> 1)], x[b][4 + e] = hi[((e & 1) << 1) | (e >> 1)];
                top = fmaxf(top, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
            }
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
        for (int b = 0; b < NB; b++) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = x[b][e] * sc;
                const _Float16 hi = (_Float16)v;
                q[0][b][e] = hi;
                sum += (float)hi;
                if constexpr (PQ == 2) q[1][b][e] = (_Float16)(v - (float)hi);
            }
            if constexpr (BIASED) {
                const float z = -72.0f * wave_xor_sum(sum);
                zero[b] = (f32x4){z, z, z, z};
            } else {
                zero[b] = (f32x4){0.f, 0.f, 0.f, 0.f};
            }
        }
    }

    f32x4 o[2 * NB];
#pragma unroll
    for (int t = 0; t < 2 * NB; t++) o[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;

    // this wave's tiles
    const int nt = (most + 31) >> 5, nw = a.nsplit * 4, gw = (int)blockIdx.x * 4 + w;
    const int lo = (int)((int64_t)gw * nt / nw), hi = (int)((int64_t)(gw + 1) * nt / nw);
    const int32_t* table = a.table + (int64_t)r * a.width;
    auto pages = [&](int t) {  // the pages of the tile's halves
        const int last = a.width - 1;
        return make_int2(table[min((32 * t) >> a.c.shift, last)], table[min((32 * t + 16) >> a.c.shift, last)]);
    };
    // this lane's place in the planes, from a half's first row
    const uint8_t* kbase = a.c.kc + ((col & 4) * 2 + (col & 3)) * (16 * NB) + g * (4 * NB);
    const uint8_t* vbase = a.c.vc + (g & 1) * (128 * NB) + col * (8 * NB);
    const uint8_t* kdbase = reinterpret_cast<const uint8_t*>(a.c.kd) + (g & 1) * (16 * NB);
    const uint8_t* vdbase = reinterpret_cast<const uint8_t*>(a.c.vd) + (g & 1) * (16 * NB);
    auto load = [&](KeyTile<NB>& x, int t, int2 pg) __attribute__((always_inline)) {
        const int p0 = __builtin_amdgcn_readfirstlane(pg.x), p1 = __builtin_amdgcn_readfirstlane(pg.y);
        const bool b0 = (unsigned)p0 >= (unsigned)a.c.pages, b1 = (unsigned)p1 >= (unsigned)a.c.pages;
        // rows of the halves' first tokens; their bytes in the code planes, 16 NB a row, and in the scales', 2 NB
        const int64_t r0 = (((int64_t)(b0 ? 0 : p0) * a.c.H + h) << a.c.shift) + ((32 * t) & (S - 1));
        const int64_t r1 = (((int64_t)(b1 ? 0 : p1) * a.c.H + h) << a.c.shift) + ((32 * t + 16) & (S - 1));
        const int64_t c0 = r0 * (16 * NB), c1 = r1 * (16 * NB), d0 = r0 * (2 * NB), d1 = r1 * (2 * NB);
        const int64_t ck = col & 8 ? c1 : c0, cv = g & 2 ? c1 : c0, dg = g & 2 ? d1 : d0;
        x.bad = g & 2 ? b1 : b0;
        load_words(kbase + ck, x.k[0]);
        load_words(kbase + ck + 4 * 16 * NB, x.k[1]);
        load_words(kdbase + dg, x.kd);
        load_words(vbase + cv, x.v);
        load_words(vdbase + dg, x.vd);
    };
    const Unpack up;
    auto compute = [&](KeyTile<NB>& x, int t) __attribute__((always_inline)) {
        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            s[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                h8 kf;
                if constexpr (BIASED) {
                    kf = up.biased(x.k[u][b]);
                } else {
                    uint32_t kw[4];
                    up.low(x.k[u][b], kw[0], kw[1]);
                    up.high(x.k[u][b], kw[2], kw[3]);
                    kf = as_h8(kw[0], kw[1], kw[2], kw[3]);
                }
                f32x4 y = zero[b];
                if constexpr (PQ == 2) y = mfma16(kf, q[1][b], y);
                y = mfma16(kf, q[0][b], y);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int n = (4 * u + e) * NB + b;  // [8][NB]
                    s[u][e] = fmaf(y[e], half_of(x.kd[n >> 1], n & 1), s[u][e]);
                }
            }
        }
        const int k0 = 32 * t + 8 * g;
        const bool edge = 32 * t + 32 > least || __any(x.bad);
        if (edge) {
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const float v = s[n >> 2][n & 3];
                s[n >> 2][n & 3] = k0 + n >= keys ? -INFINITY : x.bad ? NAN : v;
            }
            // values that no row attends count as zeros, whatever their page holds
#pragma unroll
            for (int n = 0; n < 8; n += 2) {
                const uint32_t keep = x.bad ? 0u : (k0 + n < len ? 0xffffu : 0u) | (k0 + n + 1 < len ? 0xffff0000u : 0u);
#pragma unroll
                for (int b = 0; b < NB; b++) x.vd[4 * b + (n >> 1)] &= keep;
            }
        }
        const float mx = wave_xor_max(max3f(max3f(s[0][0], s[0][1], s[0][2]), max3f(s[0][3], s[1][0], s[1][1]),
                                            fmaxf(s[1][2], s[1][3]))) * rs;
        if (__any(mx > m + RESCALE_SLACK)) {
            const float mn = fmaxf(m, mx), al = exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int b = 0; b < 2 * NB; b++) o[b] = o[b] * al;
        }
        const float mu = P_BIAS - (m == -INFINITY ? 0.0f : m);
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int n = 0; n < 8; n += 2)
            split_p<PP>(__builtin_amdgcn_exp2f(fmaf(s[n >> 2][n & 3], rs, mu)),
                        __builtin_amdgcn_exp2f(fmaf(s[n >> 2][(n & 3) + 1], rs, mu)), ph[n >> 1], pl[n >> 1], l);
        const h8 p0 = as_h8(ph[0], ph[1], ph[2], ph[3]);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                uint32_t cd[4], v[4];
                if (half) up.high(x.v[2 * b], cd[0], cd[1]), up.high(x.v[2 * b + 1], cd[2], cd[3]);
                else up.low(x.v[2 * b], cd[0], cd[1]), up.low(x.v[2 * b + 1], cd[2], cd[3]);
#pragma unroll
                for (int n = 0; n < 4; n++) v[n] = pk_mul(cd[n], x.vd[4 * b + n]);
                f32x4& acc = o[2 * b + half];
                const h8 vf = as_h8(v[0], v[1], v[2], v[3]);
                if constexpr (PV == 2) {
                    uint32_t z[4];
#pragma unroll
                    for (int n = 0; n < 4; n++) z[n] = pk_rest(cd[n], x.vd[4 * b + n], v[n]);
                    acc = mfma16(as_h8(z[0], z[1], z[2], z[3]), p0, acc);
                }
                if constexpr (PP == 2) acc = mfma16(vf, as_h8(pl[0], pl[1], pl[2], pl[3]), acc);
                acc = mfma16(vf, p0, acc);
            }
    };
    if constexpr (NB <= 4) {  // the next tile on its way while one is computed, its pages before that
        if (lo < hi) {
            KeyTile<NB> x, y;
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
    } else {  // (two tiles would not fit the registers; with one, two waves a SIMD do but at head dim 256, f32 224)
        int2 pg = lo < hi ? pages(lo) : make_int2(0, 0);
        for (int t = lo; t < hi; t++) {
            KeyTile<NB> x;
            load(x, t, pg);
            pg = pages(min(t + 1, hi - 1));
            compute(x, t);
        }
    }

    // merge the waves
    l = wave_xor_sum(l);
    if (g == 0) sml[w][col] = make_float2(m, l);
#pragma unroll
    for (int t = 0; t < 2 * NB; t++) *reinterpret_cast<f32x4*>(&so[w][col][16 * t + 4 * g]) = o[t];
    __syncthreads();
    for (int e = tid; e < 16 * (D / 4); e += 256) {
        const int rc = e / (D / 4), d = e % (D / 4) * 4, ri = first + rc;
        if (ri >= rows) break;
        float mm = -INFINITY;
#pragma unroll
        for (int s = 0; s < 4; s++) mm = fmaxf(mm, sml[s][rc].x);
        const float mu = mm == -INFINITY ? 0.0f : mm;
        float tl = 0.0f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const float f = exp2f(sml[s][rc].x - mu);
            tl += sml[s][rc].y * f;
            const f32x4 v = *reinterpret_cast<const f32x4*>(&so[s][rc][d]);
#pragma unroll
            for (int n = 0; n < 4; n++) acc[n] += v[n] * f;
        }
        if (a.nsplit == 1) {
            const int64_t row = (int64_t)(start + ri / a.G) * a.Hq + h * a.G + ri % a.G;
            const float inv = 1.0f / tl, y[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
            store4<DT>(a.out, row * D + d, y);
            if (a.lse && d == 0) a.lse[row] = tl == 0.0f ? -INFINITY : (mm - P_BIAS) * LN2 + logf(tl);
        } else {
            const int64_t row = (((int64_t)r * a.c.H + h) * a.few + ri) * a.nsplit + blockIdx.x;
            *reinterpret_cast<f32x4*>(a.part_o + row * D + d) = acc;
            if (d == 0) a.part_ml[row] = make_float2(mm, tl);
        }
    }
}

// The splits of a row, in order (the same bits every time): four output columns a thread.
// A launch of its own, 3 to 4 us: of 18 us for sixteen single rows.
template <int DT>
__global__ __launch_bounds__(256) void k_paged_combine(const PagedArgs a) {
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
    const float2* ml = a.part_ml + pr * a.nsplit;
    const float* po = a.part_o + pr * a.nsplit * D + d;
    float mm = -INFINITY, tl = 0.0f;
    for (int s = 0; s < a.nsplit; s++) mm = fmaxf(mm, ml[s].x);
    const float mu = mm == -INFINITY ? 0.0f : mm;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < a.nsplit; s++) {
        const float f = exp2f(ml[s].x - mu);
        tl += ml[s].y * f;
        const f32x4 v = *reinterpret_cast<const f32x4*>(po + (int64_t)s * D);
#pragma unroll
        for (int n = 0; n < 4; n++) acc[n] += v[n] * f;
    }
    const int64_t row = (int64_t)(start + i / a.G) * a.Hq + h * a.G + i % a.G;
    const float inv = 1.0f / tl, y[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    store4<DT>(a.out, row * D + d, y);
    if (a.lse && d == 0) a.lse[row] = tl == 0.0f ? -INFINITY : (mm - P_BIAS) * LN2 + logf(tl);
}

// ---- many rows --------------------------------------------------------------------
//
// A wave takes 32 folded rows, a workgroup 32 W of them, and keys KT at a time. The
// codes are unpacked and scaled to f16 once a workgroup, into LDS, ahead of their use:
// K as rows of D elements in the codes' order (chunk 4 b + x + 2 y of 16 bytes: part
// 2 x + y of block b, so that half x of a wave holds parts 2 x and 2 x + 1), V
// transposed, a row an element with its keys in the order in which the score product
// leaves them in a lane (keys 4 h .. 4 h + 3 of each eight in half h of the wave), so
// that P^T needs no exchange. Values are the rounded product and, but for bf16 outputs,
// what it lacks, two f16 parts; so are keys (one part: EXACT_KEYS below); probabilities
// are one but for f32 outputs. (One part shows as in k_paged_few. f16 prompts, 32 heads on 8
// of 128, take 233 us for 4096 rows and 93 for 2048; 17 % and 14 % more with probabilities
// in two parts too. bf16 rows with two of everything: 276 us for the prompt below.) Rows
// are padded by 16 bytes, which spreads 16 rows' reads over all banks.
//
// A wave alternates between a phase of products, O^T += V^T P^T of tile t and S^T of
// tile t + 1, with its share of the unpacking (V of tile t + 1, K of t + 2) in their
// shadow, and the softmax of tile t + 1. Eight waves are two groups of one wave a SIMD,
// half a turn apart: while one group's products run, the other's softmax does. The
// first group unpacks V and the second K, so that two tiles of each in LDS suffice:
// with barriers numbered as the first group passes them, it reads V(t) and K(t + 1)
// and writes V(t + 1) behind barrier 2 t + 2, the second group reads the same and
// writes K(t + 2) behind 2 t + 3; so V(t + 1) takes the place of V(t - 1), last read
// behind 2 t + 1, and K(t + 2) that of K(t), last read there too.
//
// Bound by the products, at the clock that they leave: 4096 causal rows of 32 heads of
// 128, bf16, 152 us, 900 TF/s of 1300 that a large product of matrices reaches; the clock
// falls to 1.9 GHz of 2.4. Workgroups of 256 rows keep part of their registers in scratch
// memory, inside the loop, at head dim 256 (bf16 from 224 on, f32 from 192): 2048 rows of
// 2048 keys, 32 heads on 8, at 192, 224 and 256: bf16, 98, 112 and 178 us; f16, 156, 182
// and 249; f32, 296, 437 and 624 (126 at 128). (The prompt step by step: a workgroup of 128
// rows, all in one phase, 185; packed operations and no branch in the loop, 178; 256 rows,
// 167; the two groups half a turn apart, 154; tiles asked for together at the start, output
// through LDS, 149; keys of bf16 rows in two parts up to 1024 of them, 152.)
// Fewer rows than fill the chip with 256 a workgroup run as 128 a workgroup, two a unit,
// with their keys in up to 8 splits: 512 rows behind 20000 keys, 192 us, 277 unsplit.
template <int DT, int NB, int W, int KK>
struct Many {
    static constexpr int KV = DT == TN_BF16 ? 1 : 2, Q = DT == TN_F32 ? 2 : 1, P = DT == TN_F32 ? 2 : 1;
    static constexpr int ROWS = 32 * W, GROUPS = W / 4;                // folded rows; groups of four waves
    static constexpr int D = 32 * NB, KP = 2 * D + 16;                  // K row pitch, bytes
    static constexpr int stage(int kt) { return KK * kt * KP + KV * D * (2 * kt + 16); }
    static constexpr int LDS = GROUPS == 2 ? 160 << 10 : 80 << 10;      // one or two workgroups a unit
    static constexpr int KT = NB <= 4 && 2 * stage(64) <= LDS ? 64 : 32;  // keys of a tile
    static constexpr int VP = 2 * KT + 16, KB = KT * KP, VB = D * VP, STAGE = KK * KB + KV * VB;
    static constexpr int KI = KT * 4, VI = NB * KT;                    // items: (key, part), (byte column, 16 keys)
    static constexpr int OS = DT == TN_F32 ? 4 : 2;                    // output element
    static constexpr int OP = (NB < 4 ? D : 128) * (GROUPS == 1 ? 4 : OS) + 16;  // row pitch on the way out
    static constexpr int LDS_BYTES = 2 * STAGE > ROWS * OP ? 2 * STAGE : ROWS * OP;
    static constexpr int WAVES = GROUPS == 2 || LDS_BYTES <= LDS ? 2 : 1;  // a SIMD, as launch bounds
    static_assert(KI <= 256 && VI <= 256, "an item a thread");
};

// Scales that stand in for those of a page outside the cache: NaN for keys (their
// scores are NaN), zero for values.
__device__ const uint32_t paged_stand_in[8] = {0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0, 0, 0, 0};

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
    TN_INLINE float get(int e) const {
        if constexpr (DT == TN_F32) return __uint_as_float(w[e >> 2][e & 3]);
        else return e & 1 ? El<DT == TN_F16>::hi(w[0][e >> 1]) : El<DT == TN_F16>::lo(w[0][e >> 1]);
    }
};

template <int NB>
TN_INLINE void load_scales(const uint16_t* p, uint32_t (&d)[(NB + 1) / 2]) {
    if constexpr (NB % 2 == 0) load_words(p, d);
    else {
        const TN_GLOBAL uint16_t* s = (const TN_GLOBAL uint16_t*)reinterpret_cast<uintptr_t>(p);
#pragma unroll
        for (int b = 0; b < NB; b += 2) d[b / 2] = s[b] | (b + 1 < NB ? (uint32_t)s[b + 1] << 16 : 0u);
    }
}

// Rows first .. first + ROWS of request r, whose rows start at `start` and attend
// `before` keys more than there are rows ahead of them.
template <int DT, int NB, int W, int KK>
TN_INLINE void many_tile(const PagedArgs& a, uint8_t* lds, int h, int r, int start, int rows, int first, int len,
                         int before) {
    using M = Many<DT, NB, W, KK>;
    constexpr int KT = M::KT, D = M::D, KV = M::KV, ROWS = M::ROWS;
    const int tid = threadIdx.x & 255, lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), group = w >> 2;
    const int col = lane & 31, hh = lane >> 5;
    const int S = 1 << a.c.shift;
    const int i = first + 32 * w + col, j = min(i, rows - 1) / a.G, hq = h * a.G + min(i, rows - 1) % a.G;
    const int keys = max(0, before + j + 1);
    const int least = max(0, before + min(first + 32 * w, rows - 1) / a.G + 1);  // that all of the wave's rows attend
    const int most = max(0, before + (min(first + ROWS, rows) - 1) / a.G + 1);   // that any of the workgroup's does
    // this workgroup's tiles: one split's share
    const int all_tiles = (most + KT - 1) / KT, split = blockIdx.y, ns = gridDim.y;
    const int t0 = (int)((int64_t)split * all_tiles / ns), nt = (int)((int64_t)(split + 1) * all_tiles / ns);

    // The query: step 2 b + y of the product contracts over parts y (half 0) and 2 + y
    // (half 1) of block b, so that a lane's elements of a block are eight low ones in a
    // row and eight high ones.
    h8 q[M::Q][2 * NB];
    float rs = fabsf(a.sl2);
    Eight<DT> qx[NB][2];
    auto load_q = [&]() __attribute__((always_inline)) {
        const int64_t qi = (int64_t)(start + j) * a.q_stride + (int64_t)hq * D + 8 * hh;
#pragma unroll
        for (int b = 0; b < NB; b++) qx[b][0].load(a.q, qi + 32 * b), qx[b][1].load(a.q, qi + 32 * b + 16);
    };
    auto make_q = [&]() __attribute__((always_inline)) {
        float top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(qx[b][e >> 3].get(e & 7)));
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
            for (int e = 0; e < 8; e++) {  // elements 0 2 1 3 of the part, low then high
                const float v = qx[c >> 1][e >> 2].get(4 * (c & 1) + (((e & 1) << 1) | (e >> 1 & 1))) * sc;
                const _Float16 hi = (_Float16)v;
                q[0][c][e] = hi;
                if constexpr (M::Q == 2) q[1][c][e] = (_Float16)(v - (float)hi);
            }
    };
    f32x16 o[NB], s[KT / 32];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[b][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    uint32_t ph[KT / 4], pl[KT / 4];

    // ---- this thread's part of a tile: its loads, and their way into LDS
    const int32_t* table = a.table + (int64_t)r * a.width;
    // K: (key, part), a wave's lanes on one part (their LDS rows differ); V: (16 keys, byte column)
    const int ki = tid % M::KI, key = ki % KT, part = ki / KT;
    const int place = 2 * (part & 1) + (part >> 1);
    const int vt = M::GROUPS == 1 && M::KI < 256 ? (tid + 256 - M::KI) & 255 : tid;
    const int vi = vt % M::VI, kg = vi / (16 * NB), vb = vi % (16 * NB) / 16, vcol = vi % 16;
    const bool kon = M::KI == 256 || tid < M::KI, von = M::VI == 256 || vt < M::VI;
    struct KPart { uint32_t c[NB], s[(NB + 1) / 2]; } kr;
    struct VPart { uint32_t c[4], s[8]; } vr;
    int kpage = 0, vpage = 0;
    const Unpack up;
    // (tiles past the last are the last again)
    auto kpages = [&](int t) __attribute__((always_inline)) {
        return table[min((KT * min(t, nt - 1) + key) >> a.c.shift, a.width - 1)];
    };
    auto vpages = [&](int t) __attribute__((always_inline)) {
        return table[min((KT * min(t, nt - 1) + 16 * kg) >> a.c.shift, a.width - 1)];
    };
    auto load_k = [&](KPart& x, int page, int t) __attribute__((always_inline)) {
        t = min(t, nt - 1);
        const bool bad = (unsigned)page >= (unsigned)a.c.pages;
        const int64_t row = (((int64_t)(bad ? 0 : page) * a.c.H + h) << a.c.shift) + ((KT * t + key) & (S - 1));
        load_words(a.c.kc + row * (16 * NB) + part * (4 * NB), x.c);
        load_scales<NB>(bad ? reinterpret_cast<const uint16_t*>(paged_stand_in) : a.c.kd + row * NB, x.s);
    };
    auto load_v = [&](VPart& x, int page, int t) __attribute__((always_inline)) {
        t = min(t, nt - 1);
        const bool bad = (unsigned)page >= (unsigned)a.c.pages;
        const int64_t eight =
            (((int64_t)(bad ? 0 : page) * a.c.H + h) << (a.c.shift - 3)) + (((KT * t + 16 * kg) & (S - 1)) >> 3);
        const uint8_t* p = a.c.vc + eight * (128 * NB) + (vcol * NB + vb) * 8;
        uint32_t c0[2], c1[2], s0[4], s1[4];
        load_words(p, c0);
        load_words(p + 128 * NB, c1);
        x.c[0] = c0[0], x.c[1] = c0[1], x.c[2] = c1[0], x.c[3] = c1[1];
        const uint16_t* zero = reinterpret_cast<const uint16_t*>(paged_stand_in + 4);
        load_words(bad ? zero : a.c.vd + (eight * NB + vb) * 8, s0);
        load_words(bad ? zero : a.c.vd + ((eight + 1) * NB + vb) * 8, s1);
#pragma unroll
        for (int e = 0; e < 4; e++) x.s[e] = s0[e], x.s[4 + e] = s1[e];
    };
    auto unpack_k = [&](const KPart& y, int b, int t) __attribute__((always_inline)) {  // block b of this thread's part of a row
        const uint32_t sc = (b & 1 ? y.s[b / 2] >> 16 : y.s[b / 2] & 0xffffu) * 0x10001u;
        uint32_t c[4], v[4];
        up.low(y.c[b], c[0], c[1]), up.high(y.c[b], c[2], c[3]);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = pk_mul(c[e], sc);
        uint8_t* p = lds + (t & 1) * M::STAGE + key * M::KP + (4 * b + place) * 16;
        if (kon) *reinterpret_cast<h8*>(p) = as_h8(v[0], v[1], v[2], v[3]);
        if constexpr (KK == 2) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = pk_rest(c[e], sc, v[e]);
            if (kon) *reinterpret_cast<h8*>(p + M::KB) = as_h8(v[0], v[1], v[2], v[3]);
        }
    };
    auto edge_v = [&](VPart& y, int t) __attribute__((always_inline)) {  // values that no row attends count as zeros
        if (KT * t + KT > len) {
            const int left = len - KT * t - 16 * kg;
#pragma unroll
            for (int e = 0; e < 8; e++) y.s[e] &= (2 * e < left ? 0xffffu : 0u) | (2 * e + 1 < left ? 0xffff0000u : 0u);
        }
    };
    // Half of the elements (low or high nibbles) and of the tokens of this thread's bytes.
    // Dwords 0, 1: tokens 0 .. 7; 2, 3: 8 .. 15. Half 0 holds tokens 0 .. 3 and 8 .. 11
    auto unpack_v = [&](const VPart& y, int high, int half, int t) __attribute__((always_inline)) {
        uint32_t x[4], v[4], sc[4];
        if (high) up.high(y.c[half], x[0], x[1]), up.high(y.c[2 + half], x[2], x[3]);
        else up.low(y.c[half], x[0], x[1]), up.low(y.c[2 + half], x[2], x[3]);
#pragma unroll
        for (int e = 0; e < 4; e++) sc[e] = y.s[(e >> 1) * 4 + 2 * half + (e & 1)];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = pk_mul(x[e], sc[e]);
        uint8_t* p = lds + (t & 1) * M::STAGE + KK * M::KB + (32 * vb + 16 * high + vcol) * M::VP + (2 * kg + half) * 16;
        if (von) *reinterpret_cast<h8*>(p) = as_h8(v[0], v[1], v[2], v[3]);
        if constexpr (KV == 2) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = pk_rest(x[e], sc[e], v[e]);
            if (von) *reinterpret_cast<h8*>(p + M::VB) = as_h8(v[0], v[1], v[2], v[3]);
        }
    };

    // ---- the phases
    // The products of a phase in groups of four fragments out of LDS, each group read
    // while the one before it is multiplied: PG of O^T += V^T P^T (a group is 16 keys and
    // BG blocks), then SG of S^T (XG steps of all the tile's keys).
    constexpr int BG = 4 / KV, PB = (NB + BG - 1) / BG, PG = KT / 16 * PB;
    constexpr int U = KT / 32, XG = 4 / (KK * U), SG = (2 * NB + XG - 1) / XG;
    h8 f[2][4];
    auto fetch = [&](int n, int t) __attribute__((always_inline)) {
        if (n < PG) {
            const uint8_t* st = lds + (t & 1) * M::STAGE + KK * M::KB + col * M::VP + hh * 16 + n / PB * 32;
#pragma unroll
            for (int e = 0; e < BG; e++)
#pragma unroll
                for (int p = 0; p < KV; p++)
                    if (n % PB * BG + e < NB)
                        f[n & 1][e * KV + p] =
                            *reinterpret_cast<const h8*>(st + 32 * (n % PB * BG + e) * M::VP + p * M::VB);
        } else if (n < PG + SG) {
            const uint8_t* st = lds + ((t + 1) & 1) * M::STAGE + col * M::KP + hh * 16;
#pragma unroll
            for (int x = 0; x < XG; x++)
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int p = 0; p < KK; p++)
                        if ((n - PG) * XG + x < 2 * NB)
                            f[n & 1][(x * U + u) * KK + p] = *reinterpret_cast<const h8*>(
                                st + 32 * u * M::KP + 32 * ((n - PG) * XG + x) + p * M::KB);
        }
    };
    auto multiply = [&](int n) __attribute__((always_inline)) {
        if (n < PG) {
            const int k = 4 * (n / PB);
            const h8 p0 = as_h8(ph[k], ph[k + 1], ph[k + 2], ph[k + 3]);
            const h8 p1 = M::P == 2 ? as_h8(pl[k], pl[k + 1], pl[k + 2], pl[k + 3]) : p0;
#pragma unroll
            for (int p = KV - 1; p >= 0; p--)
#pragma unroll
                for (int e = 0; e < BG; e++) {
                    const int b = n % PB * BG + e;
                    if (b >= NB) continue;
                    if (M::P == 2 && p == 0) o[b] = El<true>::mfma(f[n & 1][e * KV], p1, o[b]);
                    o[b] = El<true>::mfma(f[n & 1][e * KV + p], p0, o[b]);
                }
        } else {
#pragma unroll
            for (int x = 0; x < XG; x++) {
                const int c = (n - PG) * XG + x;
                if (c >= 2 * NB) continue;
#pragma unroll
                for (int p = KK - 1; p >= 0; p--)
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        if (M::Q == 2 && p == 0) s[u] = El<true>::mfma(f[n & 1][(x * U + u) * KK], q[M::Q - 1][c], s[u]);
                        s[u] = El<true>::mfma(f[n & 1][(x * U + u) * KK + p], q[0][c], s[u]);
                    }
            }
        }
    };
    // Groups from .. to - 1, the first of which is in registers; between their products,
    // in their shadow, this thread's part of V of tile t + 1 and K of t + 2 (role: 1 V,
    // 2 K, 3 both), then the loads of the next ones.
    auto products = [&](auto role, auto from, auto to, int t) __attribute__((always_inline)) {
        constexpr int STEPS = to.value - from.value, ROLE = role.value;
        constexpr int KW = ROLE & 2 ? NB : 0, VW = ROLE & 1 ? 4 : 0, WORK = KW + VW + (ROLE ? 1 : 0);
        if constexpr (to.value > PG) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[u][e] = 0.0f;
        }
#pragma unroll
        for (int n = from.value; n < to.value; n++) {
            __builtin_amdgcn_sched_barrier(0);
            if (n + 1 < to.value) fetch(n + 1, t);
            multiply(n);
#pragma unroll
            for (int x = (n - from.value) * WORK / STEPS; x < (n - from.value + 1) * WORK / STEPS; x++) {
                if (x < KW) unpack_k(kr, x, t + 2);
                else if (x < KW + VW) unpack_v(vr, (x - KW) >> 1, (x - KW) & 1, t + 1);
                else {
                    if constexpr (ROLE & 2) load_k(kr, kpage, t + 3), kpage = kpages(t + 4);
                    if constexpr (ROLE & 1) load_v(vr, vpage, t + 2), vpage = vpages(t + 3);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto softmax = [&](int t) __attribute__((always_inline)) {
        // the products' wait states: the compiler does not see that max3f's assembly reads their result
        __builtin_amdgcn_sched_barrier(0);
#if __HIP_DEVICE_COMPILE__
        asm volatile("s_nop 15\n\ts_nop 1");
#endif
        __builtin_amdgcn_sched_barrier(0);
        if (KT * t + KT > least) {
#pragma unroll
            for (int u = 0; u < KT / 32; u++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int k = KT * t + 32 * u + 8 * (e >> 2) + 4 * hh + (e & 3);
                    const float v = s[u][e];
                    s[u][e] = k >= keys ? -INFINITY : v;
                }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // short chains
#pragma unroll
        for (int u = 0; u < KT / 32; u++)
#pragma unroll
            for (int e = 0; e < 16; e += 2) mx4[e / 2 & 3] = max3f(mx4[e / 2 & 3], s[u][e], s[u][e + 1]);
        const float mx = xor32_max(max3f(max3f(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3])) * rs;
        if (__any(mx > m + RESCALE_SLACK)) {
            const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[b][e] *= al;
        }
        const float mu = P_BIAS - (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int u = 0; u < KT / 32; u++)
#pragma unroll
            for (int e = 0; e < 16; e += 2)
                split_p<M::P>(__builtin_amdgcn_exp2f(fmaf(s[u][e], rs, mu)),
                              __builtin_amdgcn_exp2f(fmaf(s[u][e + 1], rs, mu)), ph[8 * u + e / 2], pl[8 * u + e / 2], l);
        // computed here, not where the products take them
#if __HIP_DEVICE_COMPILE__
#pragma unroll
        for (int e = 0; e < KT / 4; e++) {
            asm volatile("" : "+v"(ph[e]));
            if constexpr (M::P == 2) asm volatile("" : "+v"(pl[e]));
        }
        asm volatile("" : "+v"(l));
#endif
    };
    auto walk = [&](auto role) __attribute__((always_inline)) {
        constexpr std::integral_constant<int, 0> BEGIN, NONE;
        constexpr std::integral_constant<int, PG> MIDDLE;
        constexpr std::integral_constant<int, PG + SG> END;
        // all that the first tiles need is asked for before any of it is waited for
        KPart k0, k1;
        VPart v0;
        int kp0 = 0, kp1 = 0, kp2 = 0, vp0 = 0, vp1 = 0;
        if constexpr (role.value & 2) kp0 = kpages(t0), kp1 = kpages(t0 + 1), kp2 = kpages(t0 + 2), kpage = kpages(t0 + 3);
        if constexpr (role.value & 1) vp0 = vpages(t0), vp1 = vpages(t0 + 1), vpage = vpages(t0 + 2);
        load_q();
        if constexpr (role.value & 2) load_k(k0, kp0, t0), load_k(k1, kp1, t0 + 1), load_k(kr, kp2, t0 + 2);
        if constexpr (role.value & 1) load_v(v0, vp0, t0), load_v(vr, vp1, t0 + 1);
        make_q();
        if constexpr (role.value & 2) {
#pragma unroll
            for (int b = 0; b < NB; b++) unpack_k(k0, b, t0), unpack_k(k1, b, t0 + 1);
        }
        if constexpr (role.value & 1) {
            edge_v(v0, t0);
#pragma unroll
            for (int x = 0; x < 4; x++) unpack_v(v0, x >> 1, x & 1, t0);
        }
        __syncthreads();
        if (role.value == 2) __syncthreads();  // half a turn behind
        fetch(PG, t0 - 1);
        products(NONE, MIDDLE, END, t0 - 1);
        for (int t = t0; t + 1 < nt; t++) {
            __syncthreads();
            if constexpr (role.value & 1) edge_v(vr, t + 1);
            softmax(t);
            fetch(0, t);
            __syncthreads();
            __builtin_amdgcn_s_setprio(1);  // the products' few instructions ahead of the other group's many
            products(role, BEGIN, END, t);
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
        softmax(nt - 1);
        fetch(0, nt - 1);
        __syncthreads();
        products(NONE, BEGIN, MIDDLE, nt - 1);
        if (role.value == 1) __syncthreads();
    };
    if (nt > t0) {
        if constexpr (M::GROUPS == 1) walk(std::integral_constant<int, 3>{});
        else if (group == 0) walk(std::integral_constant<int, 1>{});
        else walk(std::integral_constant<int, 2>{});
    }

    // out through LDS, so that a row's bytes leave together, in `type` to rows of a.out or (many_o) f32
    l = xor32_sum(l);
    uint8_t* mine = lds + w * 32 * M::OP;
    __syncthreads();
    auto leave = [&](auto type, float f) __attribute__((always_inline)) {
        constexpr int OT = type.value, SIZE = OT == TN_F32 ? 4 : 2;
#pragma unroll
        for (int b0 = 0; b0 < NB; b0 += 4) {  // four blocks at a time
            const int nb = NB - b0 < 4 ? NB - b0 : 4, pieces = nb * 2 * SIZE;  // of 16 bytes, a row
#pragma unroll
            for (int b = b0; b < b0 + nb; b++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float y[4] = {o[b][e] * f, o[b][e + 1] * f, o[b][e + 2] * f, o[b][e + 3] * f};
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
    if (M::GROUPS == 1 && ns > 1) {  // a split's part: k_paged_join's
        leave(std::integral_constant<int, TN_F32>{}, 1.0f);
        if (hh == 0 && i < rows) a.many_ml[row * ns + split] = make_float2(m, l);
    } else {
        leave(std::integral_constant<int, DT>{}, 1.0f / l);
        if (a.lse && hh == 0 && i < rows) a.lse[row] = l == 0.0f ? -INFINITY : (m - P_BIAS) * LN2 + logf(l);
    }
}

// K's parts are two, so that a score is as exact as the f32 sum. A bf16 call's rows of many
// keys make do with one, the value rounded to f16: a score is then off by 2^-12 of each
// of its products, which the output's 8 bits do not show and the lse, a mean over the
// keys, by less the more they are (a prompt of 4096 random keys: 7e-7 of its lse; one of
// 1000, in two parts, 7e-8; with one part everywhere, past 1e-6). 4096 rows of 32 heads of
// 128: 152 us; when it was 150, 144 with one part everywhere and 183 with two.
constexpr int EXACT_KEYS = 1024;

template <int DT, int NB, int W>
struct ManyLaunch {
    static constexpr int KK = DT == TN_BF16 ? 1 : 2;  // of rows of many keys
    using A = Many<DT, NB, W, 2>;
    using B = Many<DT, NB, W, KK>;
    static constexpr int LDS_BYTES = A::LDS_BYTES > B::LDS_BYTES ? A::LDS_BYTES : B::LDS_BYTES;
    static constexpr int WAVES = A::WAVES < B::WAVES ? A::WAVES : B::WAVES;
};

template <int DT, int NB, int W>
__global__ __launch_bounds__(64 * W, (ManyLaunch<DT, NB, W>::WAVES)) void k_paged_many(const PagedArgs a, int tiles) {
    using L = ManyLaunch<DT, NB, W>;
    constexpr int ROWS = 32 * W;
    __shared__ __align__(16) uint8_t lds[L::LDS_BYTES];
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
    if (first < 0 || first >= rows || rows <= a.few) return;  // few rows: k_paged_few's
    const int len = max(0, min(a.lens[r], a.max_len)), before = len - all;
    if (L::KK == 1 && before + first / a.G >= EXACT_KEYS)
        many_tile<DT, NB, W, L::KK>(a, lds, h, r, start, rows, first, len, before);
    else many_tile<DT, NB, W, 2>(a, lds, h, r, start, rows, first, len, before);
}

// The splits of k_paged_many's rows, in order: four output columns a thread.
template <int DT>
__global__ __launch_bounds__(256) void k_paged_join(const PagedArgs a, int ns) {
    const int D = 32 * a.c.nb, q4 = D / 4;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = e / q4;
    const int d = (int)(e - row * q4) * 4, t = (int)(row / a.Hq);
    if (t >= a.row_start[a.n]) return;
    int r = 0, hi = a.n;  // the row's request
    while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (a.row_start[mid] <= t) r = mid;
        else hi = mid;
    }
    const int start = start_of(a, r), c = min(rows_of(a, r, start), a.max_rows);
    if (t < start || t - start >= c || c * a.G <= a.few) return;  // (rows ahead of the first request's are no one's)
    const float2* ml = a.many_ml + row * ns;
    const float* po = a.many_o + row * ns * D + d;
    float mm = -INFINITY, tl = 0.0f;
    for (int s = 0; s < ns; s++) mm = fmaxf(mm, ml[s].x);
    const float mu = mm == -INFINITY ? 0.0f : mm;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ns; s++) {
        const float f = exp2f(ml[s].x - mu);
        tl += ml[s].y * f;
        const f32x4 v = *reinterpret_cast<const f32x4*>(po + (int64_t)s * D);
#pragma unroll
        for (int n = 0; n < 4; n++) acc[n] += v[n] * f;
    }
    const float inv = 1.0f / tl, y[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    store4<DT>(a.out, row * D + d, y);
    if (a.lse && d == 0) a.lse[row] = tl == 0.0f ? -INFINITY : (mm - P_BIAS) * LN2 + logf(tl);
}

// Splits of the keys of k_paged_few: one round of the two workgroups that a compute unit
// holds (sixteen sequences of 512 to 4096 keys, 128 workgroups a split: 17.3 us at 4
// splits, 22.4 at 6; twelve of 20000 to 40000, 96 a split: 102 us at 5, 110 at 6), of 512
// keys or more, up to eight of them of 256 (one of 1000 keys, 8 heads of 128: 8.9 us at 4,
// 10.4 at 2; eight of 100 to 3000, 4 rows each: 12.8 at 8, 13.7 at 6; but four of 1000 to
// 4000: 13.7 at 15, 11.9 at 8; one of 8000: 13.5 at 32, 12.9 at 16). Up to 512 keys are
// not worth a merge (300 keys: 5.6 us, 7.9 at 2). All measured at head dims of 64 to 128.
// At 256 (f32: 224) a unit holds one, so that 512 are two rounds: 16 sequences of 512 to
// 4096 keys, 32 heads on 8, take 36 us in bf16 (23 at 192, 26 at 224), 37 in f16, 48 in f32.
constexpr int64_t FEW_WGS = 512, FEW_KEYS = 512, FEW_MAX_SPLIT = 64;
int64_t few_most(int64_t max_len) {
    if (max_len <= FEW_KEYS) return 1;
    return std::max(std::min<int64_t>(cdiv(max_len, 256), 8), std::min(cdiv(max_len, FEW_KEYS), FEW_MAX_SPLIT));
}
int few_splits(const Pages& c, int64_t n, int64_t few, int64_t max_len) {
    const int64_t wgs = std::max<int64_t>(1, n * c.H * cdiv(few, 16));
    return (int)std::max<int64_t>(1, std::min(FEW_WGS / wgs, few_most(max_len)));
}

tn_status attn_check(const char* op, const tn_q4_cache* cache, int64_t n, int64_t tokens, int64_t Hq, int64_t max_rows,
                     int64_t max_len, Pages* c) {
    TN_TRY(paged_check(op, cache, c));
    if (n < 0 || tokens < 0 || Hq < 0 || max_rows < 0 || max_len < 0)
        return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    if (Hq % c->H)
        return fail(TN_ENOTIMPL, std::string(op) + ": " + std::to_string(Hq) + " query heads do not divide into " +
                                     std::to_string(c->H) + " key/value heads");
    // k_paged_many has up to 2 tokens * Hq + 512 n * H threads, fewer than 2^32; keys past a
    // length's last tile are still numbers of 32 bits
    if (n > 65535 || Hq > 65535 || tokens > INT32_MAX || tokens * Hq > (1 << 30) || n * c->H > (1 << 21) ||
        max_len > (1 << 30))
        return fail(TN_EVALUE, std::string(op) + ": shape too large");
    return TN_OK;
}

// Rows of its partials at most, for this call and every smaller one: no more than
// FEW_WGS workgroups of 16 rows, splits counted.
int64_t part_rows(const Pages& c, int64_t n, int64_t few, int64_t max_len) {
    const int64_t most = few_most(max_len);
    return most < 2 ? 0 : std::min(std::min<int64_t>(few, 16) * FEW_WGS, n * c.H * few * most);
}

// k_paged_many: 0 for workgroups of 256 rows (rows enough for one a unit), else the
// splits of the keys for workgroups of 128, two of which a unit holds. (us, 256 and 128 a
// workgroup, 4 heads on each of 8 of 128: bf16, 2500 rows of 2500 keys, 312 workgroups of
// 256, 75 and 77; 4000 of 4000, 145 and 161; 6000 of 6000, 307 and 334; f16, 2048 of 2048,
// 90 and 102. Unsplit, 512 rows behind 20000 keys take 277, split 192. All at head dim
// 128. Above it a unit holds one workgroup of 128 in f32, of f16 rows at 160 and 192, and of
// any type at 224 and 256; the rule counts two all the same.)
constexpr int64_t MANY_WIDE = 256, MANY_WGS = 512, MANY_MAX_SPLIT = 8;
int many_splits(const Pages& c, int64_t n, int64_t tokens, int64_t G, int64_t max_len) {
    if (tokens * G / 256 * c.H >= MANY_WIDE) return 0;
    const int64_t wgs = (tokens * G / 128 + n) * c.H;
    return (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(MANY_WGS, wgs), cdiv(max_len, 512), MANY_MAX_SPLIT}));
}
// Rows of its partials at most, for this call and every smaller one: above one split there
// are under MANY_WGS workgroups of 128 rows a split.
int64_t many_rows(const Pages& c, int64_t tokens, int64_t G, int64_t max_len) {
    const int64_t most = std::min(cdiv(max_len, 512), MANY_MAX_SPLIT);
    return most < 2 ? 0 : std::min(tokens * G * c.H * most, 2 * MANY_WGS * 128);
}

// Which kernel takes a request's rows. k_paged_few reads and unpacks the codes again for
// every 16 folded rows but starts at once and splits finely; k_paged_many fills 128 or 256
// rows, and its tiles follow one another. So k_paged_few takes all rows of a call whose
// products (tokens * Hq * max_len * D) are few, twice as many where k_paged_many has K
// and V in two parts; and of a larger call the requests of up to FEW_ROWS folded rows, if
// it is of several. (us, few and many, 8 key/value heads of 128 and 32 query heads: bf16,
// 512 rows of 1024 keys, 2.1e9, 27 and 38; 256 of 4096, 4.3e9, 47 and 42; 512 of 4096,
// 8.6e9, 85 and 57; f16: 28 and 41, 51 and 54, 92 and 84; f32: 32 and 49, 60 and 65, 110
// and 105. 4 key/value heads of 64 and 16, f16: 6 requests of 1 to 700 rows and 1000 to
// 3000 keys, 6.5e9, 55 and 71.) Its grid is as long for every request as for the longest:
// up to FEW_GRID workgroups of it.
constexpr int FEW_ROWS = 128;
constexpr int64_t FEW_WORK = 1ll << 32, FEW_GRID = 8192;

// Folded rows of a request that k_paged_few takes at most in this call; 0: it is not launched.
int64_t few_limit(const Pages& c, int dtype, int64_t n, int64_t tokens, int64_t G, int64_t max_rows, int64_t max_len) {
    const int64_t rows = max_rows * G, parts = dtype == TN_BF16 ? 1 : 2;
    // (tokens * Hq is at most 2^30, D 2^8)
    const bool little = tokens * G * c.H * 32 * c.nb <= parts * FEW_WORK / std::max<int64_t>(max_len, 1) &&
                        n * c.H * cdiv(rows, 16) <= FEW_GRID;
    return rows <= FEW_ROWS || little ? rows : n > 1 ? FEW_ROWS : 0;
}

int64_t work_rows(const Pages& c, int64_t n, int64_t tokens, int64_t G, int64_t max_rows, int64_t max_len) {
    return part_rows(c, n, max_rows * G, max_len) + (max_rows * G > FEW_ROWS ? many_rows(c, tokens, G, max_len) : 0);
}

template <int DT, int NB>
tn_status launch_at(hipStream_t st, const PagedArgs& a, int64_t tokens) {
    if (a.few) {
        const dim3 grid((unsigned)a.nsplit, (unsigned)(a.c.H * cdiv(a.few, 16)), (unsigned)a.n);
        hipLaunchKernelGGL((k_paged_few<DT, NB>), grid, dim3(256), 0, st, a);
        TN_LAUNCHED();
    }
    if ((int64_t)a.max_rows * a.G > a.few) {
        const int ns = many_splits(a.c, a.n, tokens, a.G, a.max_len);
        const bool wide = ns == 0;
        const int64_t tiles = tokens * a.G / (wide ? 256 : 128) + a.n;
        const dim3 grid((unsigned)(tiles * a.c.H), wide ? 1u : (unsigned)ns);
        if (wide) hipLaunchKernelGGL((k_paged_many<DT, NB, 8>), grid, dim3(512), 0, st, a, (int)tiles);
        else hipLaunchKernelGGL((k_paged_many<DT, NB, 4>), grid, dim3(256), 0, st, a, (int)tiles);
        TN_LAUNCHED();
        if (ns > 1) {
            const int64_t quads = tokens * a.Hq * (8 * NB);
            hipLaunchKernelGGL(k_paged_join<DT>, dim3((unsigned)cdiv(quads, 256)), dim3(256), 0, st, a, ns);
            TN_LAUNCHED();
        }
    }
    if (a.few && a.nsplit > 1) {
        const int64_t rows = (int64_t)a.n * a.c.H * a.few;
        hipLaunchKernelGGL(k_paged_combine<DT>, dim3((unsigned)cdiv(rows * (8 * NB), 256)), dim3(256), 0, st, a);
        TN_LAUNCHED();
    }
    return TN_OK;
}

template <int DT>
tn_status launch(hipStream_t st, const PagedArgs& a, int64_t tokens) {
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

int64_t tn_sdpa_paged_q4_0_work_floats(const tn_q4_cache* cache, int64_t n, int64_t tokens, int64_t Hq,
                                       int64_t max_rows, int64_t max_len) {
    Pages c;
    if (attn_check("sdpa_paged_q4_0_work_floats", cache, n, tokens, Hq, max_rows, max_len, &c) != TN_OK) return 0;
    if (!n || !tokens || !Hq || !max_rows) return 0;
    return work_rows(c, n, tokens, Hq / c.H, std::min(max_rows, tokens), max_len) * (32 * c.nb + 2);
}

tn_status tn_sdpa_paged_q4_0(void* stream, const tn_q4_cache* cache, int dtype, const void* q, int64_t q_stride,
                             int64_t tokens, int64_t Hq, int64_t n, const int32_t* row_start, const int32_t* lens,
                             const int32_t* table, int64_t width, int64_t max_rows, int64_t max_len, double scale,
                             float* work, int64_t work_floats, void* out, float* lse) {
    const char* op = "sdpa_paged_q4_0";
    PagedArgs a{};
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, "sdpa_paged_q4_0: rows must be float32, bfloat16 or float16");
    TN_TRY(attn_check(op, cache, n, tokens, Hq, max_rows, max_len, &a.c));
    const int64_t D = 32 * a.c.nb, G = Hq / a.c.H;
    if (width < 0 || width > INT32_MAX || max_len > (width << a.c.shift))
        return fail(TN_EINVAL, "sdpa_paged_q4_0: max_len " + std::to_string(max_len) + " is past what " +
                                   std::to_string(width) + " pages hold");
    if (tokens > 1 && q_stride < Hq * D) return fail(TN_EINVAL, "sdpa_paged_q4_0: the row stride is shorter than a row");
    if (tokens > 1 && q_stride > INT64_MAX / 8 / tokens)
        return fail(TN_EVALUE, "sdpa_paged_q4_0: shape too large");
    if (max_len && !a.c.pages) return fail(TN_EINVAL, "sdpa_paged_q4_0: the cache has no pages");
    const int64_t need = tn_sdpa_paged_q4_0_work_floats(cache, n, tokens, Hq, max_rows, max_len);
    if (work_floats < need)
        return fail(TN_EVALUE, "sdpa_paged_q4_0: work holds " + std::to_string(work_floats) +
                                   " floats, this call needs " + std::to_string(need));
    if (!n || !tokens || !Hq || !max_rows) return TN_OK;
    if (!q || !out || !row_start || !lens || (max_len && !table) || (need && !work))
        return fail(TN_EVALUE, "sdpa_paged_q4_0: null pointer");
    if (reinterpret_cast<uintptr_t>(work) & 15) return fail(TN_EVALUE, "sdpa_paged_q4_0: work must be 16-byte aligned");
    TN_TRY(paged_check_planes(op, a.c));
    const double sc = std::isnan(scale) ? 1.0 / std::sqrt((double)D) : scale;
    a.q = q, a.out = out, a.lse = lse, a.row_start = row_start, a.lens = lens, a.table = table;
    a.q_stride = q_stride, a.n = (int)n, a.tokens = (int)tokens, a.Hq = (int)Hq, a.G = (int)G, a.width = (int)width;
    a.max_rows = (int)std::min(max_rows, tokens), a.max_len = (int)max_len;
    a.sl2 = (float)(sc * 1.4426950408889634);
    a.few = (int)few_limit(a.c, dtype, n, tokens, G, a.max_rows, max_len);
    a.nsplit = few_splits(a.c, n, a.few, max_len);
    // f32 rows, then their pairs: the few's and the many's
    const int64_t few = part_rows(a.c, n, a.max_rows * G, max_len);
    const int64_t rows = work_rows(a.c, n, tokens, G, a.max_rows, max_len);
    a.part_o = work, a.many_o = work + few * D;
    a.part_ml = reinterpret_cast<float2*>(work + rows * D), a.many_ml = a.part_ml + few;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) return launch<TN_F32>(st, a, tokens);
    if (dtype == TN_BF16) return launch<TN_BF16>(st, a, tokens);
    return launch<TN_F16>(st, a, tokens);
}

}  // extern "C"
