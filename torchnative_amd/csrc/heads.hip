// Norms of query and key heads and the rotation of their positions, one pass.
//
// With z = x * (1 / sqrt(mean(x^2) + eps)) * weight, a head's elements turn in
// pairs, (z_i, z_{i + rot/2}) by the angle pos * inv_freq_i, and the elements
// behind rot stay. Here those are pairs as well, (rot + i, rot + (d - rot)/2 + i),
// that do not turn, so that a lane always holds pairs: a head takes 8 or 16
// lanes, which sum its squares among themselves, and nothing is read twice.
//
// The cosines and sines of a token are the same for all of its heads: a
// workgroup makes them once, into LDS. The angle is reduced to a turn in 64
// bits (its product with 1 / (2 pi) has some 2^-52 of the turns as error: at
// position 10^6 less than f32's rounding of the reduced angle).
#include <algorithm>
#include <cmath>

#include "paged.h"  // load4, store4

namespace tn {
namespace {

struct HeadArgs {
    const void *q, *k;
    void *qo, *ko;
    int64_t qs, ks, qos, kos;  // elements from a token to the next
    const float *qw, *kw, *inv_freq;
    const int32_t* pos;
    int Hq, heads, d, half;  // heads = Hq + Hkv; half = rot / 2
    float eps;
    int groups, passes;  // workgroups of a token, each of so many passes
    int nwg;
};

template <int DT>
__device__ inline float load1(const void* p, int64_t i) {
    if constexpr (DT == TN_F32) return static_cast<const float*>(p)[i];
    else {
        const uint16_t h = static_cast<const uint16_t*>(p)[i];
        return DT == TN_BF16 ? bf16_to_f32(h) : f16_bits_hw(h);
    }
}
template <int DT>
__device__ inline void store1(void* p, int64_t i, float v) {
    if constexpr (DT == TN_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = DT == TN_BF16 ? bf16_out(v) : f16_out(v);
}

// V pairs at a time (1 or 4), NC of those a lane, LH lanes a head. V = 4 takes heads
// whose turning and staying halves are multiples of four elements.
// Bound by memory where tokens are many: 8192 of 32 + 8 bf16 heads of 128 elements, 168 MB in
// and out, 38 us, 4.4 TB/s; by a launch where few (one token 1.9 us of its own).
template <int DT, int V, int LH, int NC>
__global__ __launch_bounds__(256) void k_heads(const HeadArgs a) {
    constexpr int HP = 256 / LH;  // heads of a pass
    __shared__ float2 cs[128];
    const int tid = threadIdx.x, l = tid % LH, slot = tid / LH;
    const int wg = wg_number();
    if (wg >= a.nwg) return;
    const int64_t t = wg / a.groups;
    const int h0 = wg % a.groups * a.passes * HP;
    const int half = a.half, pairs = a.d / 2, stay = pairs - half;
    if (tid < half) {
        const double turns = (double)a.pos[t] * (double)a.inv_freq[tid] * 0.15915494309189533577;
        const float angle = (float)((turns - rint(turns)) * 6.283185307179586476925);
        float s, c;
        sincosf(angle, &s, &c);
        cs[tid] = make_float2(c, s);
    }
    __syncthreads();
    for (int p = 0; p < a.passes; p++) {
        const int h = h0 + p * HP + slot;
        if (h >= a.heads) break;  // a head's lanes together
        const bool q = h < a.Hq;
        const int64_t in = q ? t * a.qs + (int64_t)h * a.d : t * a.ks + (int64_t)(h - a.Hq) * a.d;
        const int64_t out = q ? t * a.qos + (int64_t)h * a.d : t * a.kos + (int64_t)(h - a.Hq) * a.d;
        const void* src = q ? a.q : a.k;
        void* dst = q ? a.qo : a.ko;
        const float* w = q ? a.qw : a.kw;
        float x[NC][V], y[NC][V];
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int i = (c * LH + l) * V;  // the first pair
            if (i >= pairs) continue;
            const int e = i < half ? i : i + half, f = e + (i < half ? half : stay);
            if constexpr (V == 4) {
                load4<DT>(src, in + e, x[c]);
                load4<DT>(src, in + f, y[c]);
            } else {
                x[c][0] = load1<DT>(src, in + e);
                y[c][0] = load1<DT>(src, in + f);
            }
#pragma unroll
            for (int v = 0; v < V; v++) ss = ss + x[c][v] * x[c][v], ss = ss + y[c][v] * y[c][v];
        }
        if constexpr (LH == 16) ss = row16_sum(ss);
        else ss = ss + dpp_f<0xB1>(ss), ss = ss + dpp_f<0x4E>(ss), ss = ss + dpp_f<0x141>(ss);
        const float r = rms_scale(ss, a.d, a.eps);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int i = (c * LH + l) * V;
            if (i >= pairs) continue;
            const bool turn = i < half;
            const int e = turn ? i : i + half, f = e + (turn ? half : stay);
            float wx[V], wy[V];
            if constexpr (V == 4) load4<TN_F32>(w, e, wx), load4<TN_F32>(w, f, wy);
            else wx[0] = w[e], wy[0] = w[f];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float u = (x[c][v] * r) * wx[v], z = (y[c][v] * r) * wy[v];
                const float2 k = cs[turn ? i + v : 0];
                x[c][v] = turn ? u * k.x - z * k.y : u;
                y[c][v] = turn ? z * k.x + u * k.y : z;
            }
            if constexpr (V == 4) {
                store4<DT>(dst, out + e, x[c]);
                store4<DT>(dst, out + f, y[c]);
            } else {
                store1<DT>(dst, out + e, x[c][0]);
                store1<DT>(dst, out + f, y[c][0]);
            }
        }
    }
}

template <int DT, int V, int LH, int NC>
tn_status launch_at(hipStream_t st, HeadArgs& a, int64_t m) {
    const int passes = (int)cdiv(a.heads, 256 / LH);
    // a token's passes in one workgroup where tokens are many, which makes its cosines once, else
    // a workgroup each (32 + 8 bf16 heads of 128, us, one against each: 16 tokens 3.9 / 3.4, 512
    // 5.3 / 4.8, 1024 7.4 / 7.4, 2048 10.8 / 11.9, 8192 40 / 47)
    a.passes = m >= 1024 ? passes : 1;
    a.groups = (int)cdiv(passes, a.passes);
    if (m * a.groups > INT32_MAX) return fail(TN_EVALUE, "qk_norm_rope: shape too large");
    a.nwg = (int)(m * a.groups);
    hipLaunchKernelGGL((k_heads<DT, V, LH, NC>), wg_grid(a.nwg), dim3(256), 0, st, a);
    TN_LAUNCHED();
    return TN_OK;
}

template <int DT>
tn_status launch(hipStream_t st, HeadArgs& a, int64_t m) {
    if (a.half % 4 == 0 && a.d % 8 == 0) {
        if (a.d <= 64) return launch_at<DT, 4, 8, 1>(st, a, m);
        if (a.d <= 128) return launch_at<DT, 4, 16, 1>(st, a, m);
        return launch_at<DT, 4, 16, 2>(st, a, m);
    }
    return launch_at<DT, 1, 16, 8>(st, a, m);
}

}  // namespace
}  // namespace tn

using namespace tn;

extern "C" {

tn_status tn_qk_norm_rope(void* stream, int dtype, const void* q, int64_t q_stride, int64_t Hq, const void* k,
                          int64_t k_stride, int64_t Hkv, int64_t m, int64_t d, const float* q_weight,
                          const float* k_weight, double eps, const float* inv_freq, int64_t rot, const int32_t* pos,
                          void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride) {
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, "qk_norm_rope: heads must be float32, bfloat16 or float16");
    if (d < 2 || d > 256 || d % 2)
        return fail(TN_ENOTIMPL, "qk_norm_rope: head_dim " + std::to_string(d) +
                                     " is not implemented; it is even, 2 to 256");
    if (rot < 0 || rot > d || rot % 2)
        return fail(TN_EINVAL, "qk_norm_rope: " + std::to_string(rot) + " of " + std::to_string(d) +
                                   " elements cannot be rotated; an even number of them can");
    if (m < 0 || Hq < 0 || Hkv < 0) return fail(TN_EINVAL, "qk_norm_rope: bad sizes");
    if (Hq > 65535 || Hkv > 65535 || m > INT32_MAX) return fail(TN_EVALUE, "qk_norm_rope: shape too large");
    for (const int64_t s : {q_stride, q_out_stride})
        if (m > 1 && Hq && s < Hq * d) return fail(TN_EINVAL, "qk_norm_rope: the row stride is shorter than a row");
    for (const int64_t s : {k_stride, k_out_stride})
        if (m > 1 && Hkv && s < Hkv * d) return fail(TN_EINVAL, "qk_norm_rope: the row stride is shorter than a row");
    for (const int64_t s : {q_stride, q_out_stride, k_stride, k_out_stride})
        if (m > 1 && s > INT64_MAX / 8 / m) return fail(TN_EVALUE, "qk_norm_rope: shape too large");
    if (m == 0 || Hq + Hkv == 0) return TN_OK;
    if (!pos || (rot && !inv_freq) || (Hq && (!q || !q_out || !q_weight)) || (Hkv && (!k || !k_out || !k_weight)))
        return fail(TN_EVALUE, "qk_norm_rope: null pointer");
    if (m > 1 && ((Hq && q_out == q && q_out_stride != q_stride) || (Hkv && k_out == k && k_out_stride != k_stride)))
        return fail(TN_EINVAL, "qk_norm_rope: in place, a row's stride is the same on both sides");
    HeadArgs a{};
    a.q = q, a.k = k, a.qo = q_out, a.ko = k_out;
    a.qs = q_stride, a.ks = k_stride, a.qos = q_out_stride, a.kos = k_out_stride;
    a.qw = q_weight, a.kw = k_weight, a.inv_freq = inv_freq, a.pos = pos;
    a.Hq = (int)Hq, a.heads = (int)(Hq + Hkv), a.d = (int)d, a.half = (int)(rot / 2), a.eps = (float)eps;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) return launch<TN_F32>(st, a, m);
    if (dtype == TN_BF16) return launch<TN_BF16>(st, a, m);
    return launch<TN_F16>(st, a, m);
}

}  // extern "C"
