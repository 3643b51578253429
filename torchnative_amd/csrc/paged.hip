// The paged 4-bit key/value cache: the step that hands pages to requests, the
// writer and the reader of its rows (tnhip.h describes the planes).
#include "paged.h"

#include <algorithm>
#include <cmath>

#include "q8.h"

namespace tn {

tn_status paged_check(const char* op, const tn_q4_cache* cache, Pages* out) {
    const std::string name(op);
    if (!cache) return fail(TN_EVALUE, name + ": null cache");
    const int64_t S = cache->page_size, D = cache->head_dim, H = cache->n_kv_heads, P = cache->pages;
    if (S < 16 || S > 256 || (S & (S - 1)))
        return fail(TN_ENOTIMPL, name + ": page_size " + std::to_string(S) +
                                     " is not implemented; it is a power of two from 16 to 256");
    if (D < 32 || D > 256 || D % 32)
        return fail(TN_ENOTIMPL, name + ": head_dim " + std::to_string(D) +
                                     " is not implemented for a q4_0 cache; it is a multiple of 32 up to 256");
    if (H < 1 || H > 8192 || P < 0) return fail(TN_EINVAL, name + ": bad cache sizes");
    if (P > INT32_MAX / S) return fail(TN_EVALUE, name + ": a cache holds fewer than 2^31 slots");
    out->kc = cache->k_codes, out->kd = cache->k_scales, out->vc = cache->v_codes, out->vd = cache->v_scales;
    out->pages = (int)P, out->H = (int)H, out->nb = (int)(D / 32);
    out->shift = __builtin_ctzll((unsigned long long)S);
    return TN_OK;
}

tn_status paged_check_planes(const char* op, const Pages& c) {
    if (!c.pages) return TN_OK;  // nothing is read or written
    if (!c.kc || !c.kd || !c.vc || !c.vd) return fail(TN_EVALUE, std::string(op) + ": null cache plane");
    const uintptr_t all = reinterpret_cast<uintptr_t>(c.kc) | reinterpret_cast<uintptr_t>(c.kd) |
                          reinterpret_cast<uintptr_t>(c.vc) | reinterpret_cast<uintptr_t>(c.vd);
    if (all & 15) return fail(TN_EVALUE, std::string(op) + ": cache planes must be 16-byte aligned");
    return TN_OK;
}

namespace {

// ---- pages for requests -------------------------------------------------------

struct PlanArgs {
    const int32_t *fresh, *lens, *state;
    int32_t *lens_out, *table, *free_pages, *state_out, *row_start, *base, *slots, *pos;
    int n, width, shift, pages, tokens;
};

constexpr int PLAN_MAX_N = 4096;
constexpr int PLAN_THREADS = 1024;

// Inclusive sums over the workgroup's threads; `red` holds a value per wave and is
// used again only behind the caller's next barrier.
__device__ inline int64_t block_scan(int64_t v, int64_t* red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    if (lane == 63) red[w] = v;
    __syncthreads();
    int64_t before = 0;
    for (int i = 0; i < w; i++) before += red[i];
    return v + before;
}

// The slot and position of row t: its request by a search of the row starts.
__device__ inline void plan_row(const PlanArgs& a, const int32_t* starts, const int32_t* base, int t) {
    int slot = -1, p = 0;
    if (t < starts[a.n]) {
        int lo = 0, hi = a.n;  // the last request whose start is at most t and whose next one is past it
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int b = base[lo];
        if (b >= 0) {
            const int q = b + t - starts[lo];
            const int page = a.table[(int64_t)lo * a.width + (q >> a.shift)];
            if (page >= 0 && page < a.pages) {
                slot = (page << a.shift) + (q & ((1 << a.shift) - 1));
                p = q;
            }
        }
    }
    a.slots[t] = slot;
    a.pos[t] = p;
}

// One workgroup: prefix sums over the requests, pages from and to the stack, and
// the rows' slots where they are few (k_plan_rows otherwise).
__global__ __launch_bounds__(PLAN_THREADS) void k_plan(const PlanArgs a, int rows_here) {
    __shared__ int64_t red[2][PLAN_THREADS / 64];
    __shared__ int32_t s_start[PLAN_MAX_N + 1], s_base[PLAN_MAX_N];
    __shared__ int64_t s_carry[2];
    const int tid = threadIdx.x, lane = tid & 63;
    const int size = 1 << a.shift;
    const int64_t most = (int64_t)a.width << a.shift;
    auto held_of = [&](int r) { return min(max((int64_t)a.lens[r], (int64_t)0), most); };
    auto pages_of = [&](int64_t tokens) { return (int)((tokens + size - 1) >> a.shift); };

    // pages of ended requests go back onto the stack
    int64_t count = min(max(a.state[0], 0), a.pages);
    for (int r0 = 0; r0 < a.n; r0 += PLAN_THREADS) {
        const int r = r0 + tid;
        const bool ended = r < a.n && a.fresh[r] < 0;
        const int give = ended ? pages_of(held_of(r)) : 0;
        const int64_t end = block_scan(give, red[0]);
        if (tid == PLAN_THREADS - 1) s_carry[0] = end;
        const int64_t at = count + end - give;
        // a few pages by the request's own lane, more by its wave
        for (int j = 0; j < min(give, 4); j++)
            if (at + j < a.pages) a.free_pages[at + j] = a.table[(int64_t)r * a.width + j];
        uint64_t long_ones = __ballot(give > 4);
        while (long_ones) {
            const int src = __ffsll((unsigned long long)long_ones) - 1;
            long_ones &= long_ones - 1;
            const int g = __shfl(give, src);
            const int64_t to = __shfl(at, src);
            const int64_t row = (int64_t)(r - lane + src) * a.width;
            for (int j = 4 + lane; j < g; j += 64)
                if (to + j < a.pages) a.free_pages[to + j] = a.table[row + j];
        }
        __syncthreads();
        count += s_carry[0];
        __syncthreads();
    }
    count = min(count, (int64_t)a.pages);

    // each request's rows and pages
    int64_t rows = 0, taken = 0, lacking = 0, used = 0;
    if (tid == 0) s_start[0] = 0, a.row_start[0] = 0;
    for (int r0 = 0; r0 < a.n; r0 += PLAN_THREADS) {
        const int r = r0 + tid;
        int64_t len = 0, add = 0;
        bool ended = false;
        if (r < a.n) {
            const int f = a.fresh[r];
            ended = f < 0;
            add = max(f, 0);
            len = ended ? 0 : held_of(r);
        }
        const int held = pages_of(len);
        const int need = (int)min((int64_t)INT32_MAX, ((len + add + size - 1) >> a.shift) - held);
        const int64_t row_end = rows + block_scan(add, red[0]);
        const bool bad = len + add > most || row_end > a.tokens;
        const int want = bad ? 0 : need;
        const int64_t asked = taken + block_scan(want, red[1]);
        const bool ok = !bad && (need == 0 || asked <= count);
        const int64_t first = asked - want;
        if (tid == PLAN_THREADS - 1) s_carry[0] = row_end, s_carry[1] = asked;
        if (r < a.n) {
            a.lens_out[r] = (int)(ok ? len + add : len);
            a.base[r] = s_base[r] = ok ? (int)len : -1;
            a.row_start[r + 1] = s_start[r + 1] = (int)min(row_end, (int64_t)a.tokens);
        }
        const int get = ok && r < a.n ? need : 0;
        if (r < a.n && !ok) lacking += need;
        if (get) used = max(used, asked);
        for (int j = 0; j < min(get, 4); j++)
            a.table[(int64_t)r * a.width + held + j] = a.free_pages[count - 1 - (first + j)];
        uint64_t long_ones = __ballot(get > 4);
        while (long_ones) {
            const int src = __ffsll((unsigned long long)long_ones) - 1;
            long_ones &= long_ones - 1;
            const int g = __shfl(get, src), h = __shfl(held, src);
            const int64_t from = __shfl(first, src);
            const int64_t row = (int64_t)(r - lane + src) * a.width + h;
            for (int j = 4 + lane; j < g; j += 64) a.table[row + j] = a.free_pages[count - 1 - (from + j)];
        }
        __syncthreads();
        rows = s_carry[0], taken = s_carry[1];
        __syncthreads();
    }
    // `asked` of the last request that took pages is what left the stack
    const int64_t lack = block_scan(lacking, red[0]);
#pragma unroll
    for (int o = 32; o; o >>= 1) used = max(used, (int64_t)__shfl_xor(used, o));
    __syncthreads();
    if (lane == 0) red[1][tid >> 6] = used;
    __syncthreads();
    if (tid == PLAN_THREADS - 1) {
        for (int i = 0; i < PLAN_THREADS / 64; i++) used = max(used, red[1][i]);
        a.state_out[0] = (int)(count - used);
        a.state_out[1] = (int)min(lack, (int64_t)INT32_MAX);
    }
    if (rows_here)
        for (int t = tid; t < a.tokens; t += PLAN_THREADS) plan_row(a, s_start, s_base, t);
}

// The slots of many rows: the row starts in LDS, a row a thread.
__global__ __launch_bounds__(256) void k_plan_rows(const PlanArgs a) {
    __shared__ int32_t s_start[PLAN_MAX_N + 1];
    for (int i = threadIdx.x; i <= a.n; i += 256) s_start[i] = a.row_start[i];
    __syncthreads();
    for (int t = blockIdx.x * 256 + threadIdx.x; t < a.tokens; t += gridDim.x * 256) plan_row(a, s_start, a.base, t);
}

// ---- rows into the cache and back ------------------------------------------------

constexpr float KV_MAX_SCALE = 8188.0f;  // 8 * 8188 = 65504, f16's largest

// Four lanes a block: lane g holds elements 4g .. 4g+3 and 16+4g .. 16+4g+3, so
// that it makes bytes 4g .. 4g+3 of the block. The block's extreme is the first
// element of the largest size (BlockQ4_0::from_float, k_quants.rs:241-277).
template <int DT>
__device__ inline uint32_t quantise_part(const void* x, int64_t at, int g, uint16_t* scale) {
    float lo[4], hi[4];
    load4<DT>(x, at + 4 * g, lo);
    load4<DT>(x, at + 16 + 4 * g, hi);
    float a = 0.0f, top = 0.0f;
    int idx = 32;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float v = j < 4 ? lo[j & 3] : hi[j & 3];
        if (a < fabsf(v)) a = fabsf(v), top = v, idx = (j < 4 ? 0 : 12) + 4 * g + j;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float a2 = __shfl_xor(a, o, 4), t2 = __shfl_xor(top, o, 4);
        const int i2 = __shfl_xor(idx, o, 4);
        if (a < a2 || (a == a2 && i2 < idx)) a = a2, top = t2, idx = i2;
    }
    const float d = fminf(fmaxf(top / -8.0f, -KV_MAX_SCALE), KV_MAX_SCALE);
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    *scale = f16_out(d);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int q0 = min(sat_u8(lo[j] * id + 8.5f), 15), q1 = min(sat_u8(hi[j] * id + 8.5f), 15);
        w |= (uint32_t)(q0 | (q1 << 4)) << (8 * j);
    }
    return w;
}

struct RowArgs {
    Pages c;
    const void *k, *v;
    void *ko, *vo;
    int64_t stride;
    const int32_t* slots;
    int64_t items;  // quarter blocks of K, and as many of V
};

// A quarter block a lane; blockIdx.y: K or V.
template <int DT>
__global__ __launch_bounds__(256) void k_append(const RowArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (item >= a.items) return;  // items is a multiple of 4: blocks stay whole
    const int g = (int)(item & 3), nb = a.c.nb;
    const int64_t blk = item >> 2;
    const int b = (int)(blk % nb);
    const int64_t th = blk / nb;
    const int h = (int)(th % a.c.H);
    const int64_t t = th / a.c.H;
    const int slot = a.slots[t];
    if (slot < 0 || (slot >> a.c.shift) >= a.c.pages) return;
    const int64_t ph = (int64_t)(slot >> a.c.shift) * a.c.H + h;
    const int o = slot & ((1 << a.c.shift) - 1);
    uint16_t d;
    const uint32_t w = quantise_part<DT>(blockIdx.y ? a.v : a.k, t * a.stride + ((int64_t)h * nb + b) * 32, g, &d);
    if (blockIdx.y == 0) {
        const int64_t row = (ph << a.c.shift) + o;
        *reinterpret_cast<uint32_t*>(a.c.kc + row * (16 * nb) + (g * nb + b) * 4) = w;
        if (g == 0) a.c.kd[row * nb + b] = d;
    } else {
        const int64_t group = (ph << (a.c.shift - 3)) + (o >> 3);
        uint8_t* p = a.c.vc + group * (128 * nb) + v_place(o & 7);
#pragma unroll
        for (int j = 0; j < 4; j++) p[((4 * g + j) * nb + b) * 8] = (uint8_t)(w >> (8 * j));
        if (g == 0) a.c.vd[(group * nb + b) * 8 + (o & 7)] = d;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_read(const RowArgs a) {
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (item >= a.items) return;
    const int g = (int)(item & 3), nb = a.c.nb;
    const int64_t blk = item >> 2;
    const int b = (int)(blk % nb);
    const int64_t th = blk / nb;
    const int h = (int)(th % a.c.H);
    const int slot = a.slots[th / a.c.H];
    float lo[4], hi[4];
    if (slot < 0 || (slot >> a.c.shift) >= a.c.pages) {
#pragma unroll
        for (int j = 0; j < 4; j++) lo[j] = hi[j] = NAN;
    } else {
        const int64_t ph = (int64_t)(slot >> a.c.shift) * a.c.H + h;
        const int o = slot & ((1 << a.c.shift) - 1);
        uint32_t w = 0;
        uint16_t d;
        if (blockIdx.y == 0) {
            const int64_t row = (ph << a.c.shift) + o;
            w = *reinterpret_cast<const uint32_t*>(a.c.kc + row * (16 * nb) + (g * nb + b) * 4);
            d = a.c.kd[row * nb + b];
        } else {
            const int64_t group = (ph << (a.c.shift - 3)) + (o >> 3);
            const uint8_t* p = a.c.vc + group * (128 * nb) + v_place(o & 7);
#pragma unroll
            for (int j = 0; j < 4; j++) w |= (uint32_t)p[((4 * g + j) * nb + b) * 8] << (8 * j);
            d = a.c.vd[(group * nb + b) * 8 + (o & 7)];
        }
        const float s = f16_bits_hw(d);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            lo[j] = (float)((int)((w >> (8 * j)) & 15) - 8) * s;
            hi[j] = (float)((int)((w >> (8 * j + 4)) & 15) - 8) * s;
        }
    }
    void* out = blockIdx.y ? a.vo : a.ko;
    store4<DT>(out, blk * 32 + 4 * g, lo);
    store4<DT>(out, blk * 32 + 16 + 4 * g, hi);
}

tn_status row_check(const char* op, const tn_q4_cache* cache, int dtype, int64_t m, RowArgs* a) {
    TN_TRY(paged_check(op, cache, &a->c));
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, std::string(op) + ": rows must be float32, bfloat16 or float16");
    if (m < 0) return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    a->items = m * a->c.H * a->c.nb * 4;
    if (m > INT32_MAX || cdiv(a->items, 256) > WG_ROW * 2)
        return fail(TN_EVALUE, std::string(op) + ": shape too large");
    return TN_OK;
}

}  // namespace
}  // namespace tn

using namespace tn;

extern "C" {

tn_status tn_paged_plan(void* stream, int64_t n, const int32_t* fresh, const int32_t* lens, int32_t* lens_out,
                        int32_t* table, int64_t width, int64_t page_size, int32_t* free_pages, int64_t pages,
                        const int32_t* state, int32_t* state_out, int64_t tokens, int32_t* row_start, int32_t* base,
                        int32_t* slots, int32_t* pos) {
    const char* op = "paged_plan";
    tn_q4_cache shape{};
    shape.pages = pages, shape.page_size = page_size, shape.n_kv_heads = 1, shape.head_dim = 32;
    Pages c;
    TN_TRY(paged_check(op, &shape, &c));
    if (n < 0 || width < 0 || tokens < 0) return fail(TN_EINVAL, "paged_plan: bad sizes");
    if (n > PLAN_MAX_N)
        return fail(TN_ENOTIMPL, "paged_plan: " + std::to_string(n) + " requests in one step; at most " +
                                     std::to_string(PLAN_MAX_N) + " are implemented");
    if (width > INT32_MAX / page_size || tokens > INT32_MAX) return fail(TN_EVALUE, "paged_plan: shape too large");
    if (!row_start || !state || !state_out || (n && (!fresh || !lens || !lens_out || !base)) ||
        (n && width && !table) || (pages && !free_pages) || (tokens && (!slots || !pos)))
        return fail(TN_EVALUE, "paged_plan: null pointer");
    PlanArgs a{};
    a.fresh = fresh, a.lens = lens, a.state = state, a.lens_out = lens_out, a.table = table;
    a.free_pages = free_pages, a.state_out = state_out, a.row_start = row_start, a.base = base;
    a.slots = slots, a.pos = pos;
    a.n = (int)n, a.width = (int)width, a.shift = c.shift, a.pages = (int)pages, a.tokens = (int)tokens;
    const bool here = tokens <= 4 * PLAN_THREADS;
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(k_plan, dim3(1), dim3(PLAN_THREADS), 0, st, a, (int)here);
    TN_LAUNCHED();
    if (!here) {
        hipLaunchKernelGGL(k_plan_rows, dim3((unsigned)std::min<int64_t>(cdiv(tokens, 256), 1024)), dim3(256), 0, st, a);
        TN_LAUNCHED();
    }
    return TN_OK;
}

tn_status tn_kv_append_q4_0(void* stream, const tn_q4_cache* cache, int dtype, const void* k, const void* v, int64_t m,
                            int64_t stride, const int32_t* slots) {
    const char* op = "kv_append_q4_0";
    RowArgs a{};
    TN_TRY(row_check(op, cache, dtype, m, &a));
    if (m > 1 && stride < (int64_t)a.c.H * a.c.nb * 32)
        return fail(TN_EINVAL, "kv_append_q4_0: the row stride is shorter than a row");
    if (m > 1 && stride > INT64_MAX / 8 / m) return fail(TN_EVALUE, "kv_append_q4_0: shape too large");
    if (m == 0) return TN_OK;
    if (!k || !v || !slots) return fail(TN_EVALUE, "kv_append_q4_0: null pointer");
    TN_TRY(paged_check_planes(op, a.c));
    a.k = k, a.v = v, a.stride = stride, a.slots = slots;
    const dim3 grid((unsigned)cdiv(a.items, 256), 2);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) hipLaunchKernelGGL(k_append<TN_F32>, grid, dim3(256), 0, st, a);
    else if (dtype == TN_BF16) hipLaunchKernelGGL(k_append<TN_BF16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_append<TN_F16>, grid, dim3(256), 0, st, a);
    TN_LAUNCHED();
    return TN_OK;
}

tn_status tn_kv_read_q4_0(void* stream, const tn_q4_cache* cache, const int32_t* slots, int64_t m, int dtype, void* k,
                          void* v) {
    const char* op = "kv_read_q4_0";
    RowArgs a{};
    TN_TRY(row_check(op, cache, dtype, m, &a));
    if (m == 0) return TN_OK;
    if (!k || !v || !slots) return fail(TN_EVALUE, "kv_read_q4_0: null pointer");
    TN_TRY(paged_check_planes(op, a.c));
    a.ko = k, a.vo = v, a.slots = slots;
    const dim3 grid((unsigned)cdiv(a.items, 256), 2);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == TN_F32) hipLaunchKernelGGL(k_read<TN_F32>, grid, dim3(256), 0, st, a);
    else if (dtype == TN_BF16) hipLaunchKernelGGL(k_read<TN_BF16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_read<TN_F16>, grid, dim3(256), 0, st, a);
    TN_LAUNCHED();
    return TN_OK;
}

}  // extern "C"
