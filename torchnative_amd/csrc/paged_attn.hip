// Attention of ragged rows over the paged 4-bit cache (tnhip.h describes the
// planes and the rows).
#include "paged.h"

#include <algorithm>
#include <cmath>

#include "attn_common.h"

namespace tn {
namespace {

struct PagedArgs {
    Pages c;
    const void* q;
    void* out;
    float* lse;  // nullable
    const int32_t *row_start, *lens, *table;
    int64_t q_stride;
    int n, Hq, G, width, tokens, max_rows, max_len;  // G = Hq / H
    float sl2;                                      // scale * log2(e)
};

// One workgroup a (row, query head).
template <int DT>
__global__ __launch_bounds__(256) void k_paged_plain(const PagedArgs a) {
    __shared__ float sq[256], sp[256], red[4];
    const int t = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x;
    if (t >= a.row_start[a.n]) return;
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int r = lo, j = t - a.row_start[r], c = a.row_start[r + 1] - a.row_start[r];
    if (j >= a.max_rows) return;
    const int len = max(0, min(a.lens[r], a.max_len)), keys = max(0, len - c + j + 1);
    const int nb = a.c.nb, D = 32 * nb, h = hq / a.G;
    const int S = 1 << a.c.shift;
    auto qv = [&](int d) {
        const int64_t i = t * a.q_stride + (int64_t)hq * D + d;
        if constexpr (DT == TN_F32) return static_cast<const float*>(a.q)[i];
        else if constexpr (DT == TN_BF16) return bf16_to_f32(static_cast<const uint16_t*>(a.q)[i]);
        else return f16_bits_hw(static_cast<const uint16_t*>(a.q)[i]);
    };
    if (tid < D) sq[tid] = qv(tid);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int k0 = 0; k0 < keys; k0 += 256) {
        const int key = k0 + tid;
        float s = -INFINITY;
        __syncthreads();
        if (key < keys) {
            const int page = a.table[(int64_t)r * a.width + (key >> a.c.shift)];
            if (page < 0 || page >= a.c.pages) {
                s = NAN;
            } else {
                const int64_t row = (((int64_t)page * a.c.H + h) << a.c.shift) + (key & (S - 1));
                s = 0.0f;
                for (int b = 0; b < nb; b++) {
                    float x = 0.0f;
                    for (int g = 0; g < 4; g++) {
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(a.c.kc + row * (16 * nb) + (g * nb + b) * 4);
                        for (int e = 0; e < 4; e++) {
                            x += sq[32 * b + 4 * g + e] * (float)((int)((w >> (8 * e)) & 15) - 8);
                            x += sq[32 * b + 16 + 4 * g + e] * (float)((int)((w >> (8 * e + 4)) & 15) - 8);
                        }
                    }
                    s += x * f16_bits_hw(a.c.kd[row * nb + b]);
                }
                s *= a.sl2;
            }
        }
        // a NaN score has to reach the maximum
        float mx = s;
        for (int i = 32; i; i >>= 1) {
            const float u = __shfl_xor(mx, i);
            mx = mx != mx || u != u ? NAN : fmaxf(mx, u);
        }
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        float mn = m;
        for (int i = 0; i < 4; i++) mn = mn != mn || red[i] != red[i] ? NAN : fmaxf(mn, red[i]);
        const float mu = mn == -INFINITY ? 0.0f : mn, al = exp2f(m - mu);
        m = mn;
        sp[tid] = exp2f(s - mu);
        __syncthreads();
        l *= al;
        o *= al;
        for (int i = 0; i < min(256, keys - k0); i++) {
            l += sp[i];
            if (tid < D) {
                const int kk = k0 + i, page = a.table[(int64_t)r * a.width + (kk >> a.c.shift)];
                if (page < 0 || page >= a.c.pages) continue;
                const int off = kk & (S - 1), b = tid / 32, e = tid % 32;
                const int64_t group = (((int64_t)page * a.c.H + h) << (a.c.shift - 3)) + (off >> 3);
                const int w = a.c.vc[group * (128 * nb) + ((e & 15) * nb + b) * 8 + v_place(off & 7)];
                o += sp[i] * ((float)((e < 16 ? w & 15 : w >> 4) - 8) * f16_bits_hw(a.c.vd[(group * nb + b) * 8 + (off & 7)]));
            }
        }
    }
    const int64_t at = (int64_t)t * a.Hq + hq;
    if (tid < D) {
        const float y = o / l;
        if constexpr (DT == TN_F32) static_cast<float*>(a.out)[at * D + tid] = y;
        else static_cast<uint16_t*>(a.out)[at * D + tid] = DT == TN_BF16 ? bf16_out(y) : f16_out(y);
    }
    if (a.lse && tid == 0) a.lse[at] = m == -INFINITY ? -INFINITY : m * LN2 + logf(l);
}

tn_status attn_check(const char* op, const tn_q4_cache* cache, int64_t n, int64_t tokens, int64_t Hq, int64_t max_rows,
                     int64_t max_len, Pages* c) {
    TN_TRY(paged_check(op, cache, c));
    if (n < 0 || tokens < 0 || Hq < 0 || max_rows < 0 || max_len < 0)
        return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    if (Hq % c->H)
        return fail(TN_ENOTIMPL, std::string(op) + ": " + std::to_string(Hq) + " query heads do not divide into " +
                                     std::to_string(c->H) + " key/value heads");
    if (n > 65535 || Hq > 65535 || tokens > INT32_MAX || tokens * Hq > INT32_MAX || max_len > INT32_MAX)
        return fail(TN_EVALUE, std::string(op) + ": shape too large");
    return TN_OK;
}

int64_t work_floats(const Pages& c, int64_t n, int64_t tokens, int64_t Hq, int64_t max_rows, int64_t max_len) {
    return 0;
}

}  // namespace
}  // namespace tn

using namespace tn;

extern "C" {

int64_t tn_sdpa_paged_q4_0_work_floats(const tn_q4_cache* cache, int64_t n, int64_t tokens, int64_t Hq,
                                       int64_t max_rows, int64_t max_len) {
    Pages c;
    if (attn_check("sdpa_paged_q4_0_work_floats", cache, n, tokens, Hq, max_rows, max_len, &c) != TN_OK) return 0;
    return work_floats(c, n, tokens, Hq, max_rows, max_len);
}

tn_status tn_sdpa_paged_q4_0(void* stream, const tn_q4_cache* cache, int dtype, const void* q, int64_t q_stride,
                             int64_t tokens, int64_t Hq, int64_t n, const int32_t* row_start, const int32_t* lens,
                             const int32_t* table, int64_t width, int64_t max_rows, int64_t max_len, double scale,
                             float* work, int64_t work_floats_given, void* out, float* lse) {
    const char* op = "sdpa_paged_q4_0";
    PagedArgs a{};
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, "sdpa_paged_q4_0: rows must be float32, bfloat16 or float16");
    TN_TRY(attn_check(op, cache, n, tokens, Hq, max_rows, max_len, &a.c));
    const int64_t D = 32 * a.c.nb;
    if (width < 0 || width > INT32_MAX || max_len > (width << a.c.shift))
        return fail(TN_EINVAL, "sdpa_paged_q4_0: max_len " + std::to_string(max_len) + " is past what " +
                                   std::to_string(width) + " pages hold");
    if (tokens > 1 && q_stride < Hq * D) return fail(TN_EINVAL, "sdpa_paged_q4_0: the row stride is shorter than a row");
    if (tokens > 1 && q_stride > INT64_MAX / 8 / tokens)
        return fail(TN_EVALUE, "sdpa_paged_q4_0: shape too large");
    const int64_t need = work_floats(a.c, n, tokens, Hq, max_rows, max_len);
    if (work_floats_given < need)
        return fail(TN_EVALUE, "sdpa_paged_q4_0: work holds " + std::to_string(work_floats_given) +
                                   " floats, this call needs " + std::to_string(need));
    if (!n || !tokens || !Hq || !max_rows) return TN_OK;
    if (!q || !out || !row_start || !lens || (max_len && !table) || (need && !work))
        return fail(TN_EVALUE, "sdpa_paged_q4_0: null pointer");
    if (reinterpret_cast<uintptr_t>(work) & 15) return fail(TN_EVALUE, "sdpa_paged_q4_0: work must be 16-byte aligned");
    TN_TRY(paged_check_planes(op, a.c));
    const double sc = std::isnan(scale) ? 1.0 / std::sqrt((double)D) : scale;
    a.q = q, a.out = out, a.lse = lse, a.row_start = row_start, a.lens = lens, a.table = table;
    a.q_stride = q_stride, a.n = (int)n, a.Hq = (int)Hq, a.G = (int)(Hq / a.c.H), a.width = (int)width;
    a.tokens = (int)tokens, a.max_rows = (int)std::min<int64_t>(max_rows, INT32_MAX), a.max_len = (int)max_len;
    a.sl2 = (float)(sc * 1.4426950408889634);
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)tokens, (unsigned)Hq);
    if (dtype == TN_F32) hipLaunchKernelGGL(k_paged_plain<TN_F32>, grid, dim3(256), 0, st, a);
    else if (dtype == TN_BF16) hipLaunchKernelGGL(k_paged_plain<TN_BF16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_paged_plain<TN_F16>, grid, dim3(256), 0, st, a);
    TN_LAUNCHED();
    return TN_OK;
}

}  // extern "C"
