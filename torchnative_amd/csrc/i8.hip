// Rows in 8-bit integers under one scale a row, and the linear over them
// (tnhip.h: tn_i8_*).
//
// Both operands are int8 over the whole of K, so the product is one exact
// integer sum an output, on the int8 matrix core, and its only roundings are the
// epilogue's: y = ((float)sum * w_scale) * a_scale (+ bias). A row's bits thus
// do not depend on the tile, the split or the rows around it.
#include <algorithm>
#include <cmath>

#include "paged.h"  // load4

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

// Four codes in a dword of four values under 1 / scale; a value that is not finite leaves 0.
__device__ inline uint32_t codes4(const float (&v)[4], float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float c = fminf(fmaxf(rintf(v[j] * inv), -127.0f), 127.0f);
        w |= ((uint32_t)(int)c & 0xffu) << (8 * j);
    }
    return w;
}

// A workgroup of T threads a row.
template <int DT, int T>
__global__ __launch_bounds__(256) void k_i8_rows(const void* __restrict__ x, int m, int k, int8_t* __restrict__ codes,
                                                 float* __restrict__ scales) {
    constexpr int RW = 256 / T;
    __shared__ float red[4];
    __shared__ int bad[4];
    const int tid = threadIdx.x % T, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * RW + threadIdx.x / T;
    const bool on = row < m;
    const int64_t at = (on ? row : 0) * k;
    const int pitch = (int)pitch_of(k);
    float top = 0.0f;
    int odd = 0;
    auto take = [&](float v) {
        const float a = fabsf(v);
        if (a < INFINITY) top = fmaxf(top, a);
        else odd = 1;
    };
    auto load = [&](int i, float (&v)[4]) {  // elements i .. i + 3, zeros behind the row
        if (i + 4 <= k) load4<DT>(x, at + i, v);
        else {
            float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int j = 0; j < 4; j++)
                if (i + j < k) {
                    if constexpr (DT == TN_F32) u[j] = static_cast<const float*>(x)[at + i + j];
                    else {
                        const uint16_t h = static_cast<const uint16_t*>(x)[at + i + j];
                        u[j] = DT == TN_BF16 ? bf16_to_f32(h) : f16_bits_hw(h);
                    }
                }
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = u[j];
        }
    };
    for (int i = 4 * tid; i < k; i += 4 * T) {
        float v[4];
        load(i, v);
#pragma unroll
        for (int j = 0; j < 4; j++) take(v[j]);
    }
    top = xor32_max(xor16_max(row16_max(top)));
    odd = __any(odd);
    if constexpr (T > 64) {
        if (lane == 0) red[w] = top, bad[w] = odd;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        odd = bad[0] | bad[1] | bad[2] | bad[3];
    }
    if (!on) return;
    const float s = scale_of(top), inv = odd || s == 0.0f ? 0.0f : 1.0f / s;
    if (tid == 0) scales[row] = odd ? NAN : s;
    uint32_t* out = reinterpret_cast<uint32_t*>(codes + row * pitch);
    for (int i = 4 * tid; i < pitch; i += 4 * T) {
        float v[4];
        load(i, v);
        out[i / 4] = odd ? 0u : codes4(v, inv);
    }
}

struct MmArgs {
    Codes a, w;
    const float* bias;  // nullable
    void* y;
    int m, n, pitch, y_dtype;
};

__device__ inline void put(const MmArgs& a, int row, int col, int sum) {
    float v = ((float)sum * a.w.s[col]) * a.a.s[row];
    if (a.bias) v = v + a.bias[col];
    const int64_t i = (int64_t)row * a.n + col;
    if (a.y_dtype == TN_F32) static_cast<float*>(a.y)[i] = v;
    else static_cast<uint16_t*>(a.y)[i] = a.y_dtype == TN_BF16 ? bf16_out(v) : f16_out(v);
}

__device__ __attribute__((always_inline)) inline i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
#else
    (void)a, (void)b;
    return c;
#endif
}

// A wave a 16 x 16 tile, its operands straight from memory.
__global__ __launch_bounds__(256) void k_i8_tile(const MmArgs a, int mt, int64_t tiles) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int64_t tile = (int64_t)wg_number() * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int m0 = (int)(tile % mt) * 16, n0 = (int)(tile / mt) * 16;
    const int8_t* pa = a.a.c + (int64_t)min(m0 + c, a.m - 1) * a.pitch + 16 * g;
    const int8_t* pw = a.w.c + (int64_t)min(n0 + c, a.n - 1) * a.pitch + 16 * g;
    i32x4 acc = {0, 0, 0, 0};
    for (int k = 0; k < a.pitch; k += 64)
        acc = mfma_i8(*reinterpret_cast<const i32x4*>(pa + k), *reinterpret_cast<const i32x4*>(pw + k), acc);
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (m0 + 4 * g + r < a.m && n0 + c < a.n) put(a, m0 + 4 * g + r, n0 + c, acc[r]);
}

tn_status matmul(hipStream_t st, const MmArgs& a) {
    const int64_t mt = cdiv(a.m, 16), tiles = mt * cdiv(a.n, 16);
    hipLaunchKernelGGL(k_i8_tile, wg_grid(cdiv(tiles, 4)), dim3(256), 0, st, a, (int)mt, tiles);
    TN_LAUNCHED();
    return TN_OK;
}

template <int DT>
void rows_launch(hipStream_t st, const void* x, int m, int k, int8_t* codes, float* scales) {
    if (k <= 1024)
        hipLaunchKernelGGL((k_i8_rows<DT, 64>), dim3((unsigned)cdiv(m, 4)), dim3(256), 0, st, x, m, k, codes, scales);
    else hipLaunchKernelGGL((k_i8_rows<DT, 256>), dim3((unsigned)m), dim3(256), 0, st, x, m, k, codes, scales);
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

int64_t work_bytes(int64_t m, int64_t k) { return m * pitch_of(k) + (m * 4 + 15) / 16 * 16; }

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
    if (unaligned(w) || unaligned(work)) return fail(TN_EVALUE, "i8_linear: codes and work must be 16-byte aligned");
    int8_t* codes = static_cast<int8_t*>(work);
    float* scales = reinterpret_cast<float*>(codes + m * pitch_of(k));
    TN_TRY(quantize((hipStream_t)stream, x, x_dtype, m, k, codes, scales));
    MmArgs p{{codes, scales}, {w, w_scales}, bias, y, (int)m, (int)n, (int)pitch_of(k), y_dtype};
    return matmul((hipStream_t)stream, p);
}

}  // extern "C"
