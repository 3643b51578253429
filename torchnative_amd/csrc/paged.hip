// The paged 4-bit key/value cache: the step that hands pages to requests, the
// writer and the reader of its rows (tnhip.h describes the planes).
#include "paged.h"

#include <algorithm>
#include <cmath>

#include "q8.h"

namespace tn {
namespace {

template <class Cache, class Planes>
tn_status check_sizes(const char* op, const char* format, const Cache* cache, Planes* out) {
    const std::string name(op);
    if (!cache) return fail(TN_EVALUE, name + ": null cache");
    const int64_t S = cache->page_size, D = cache->head_dim, H = cache->n_kv_heads, P = cache->pages;
    if (S < 16 || S > 256 || (S & (S - 1)))
        return fail(TN_ENOTIMPL, name + ": page_size " + std::to_string(S) +
                                     " is not implemented; it is a power of two from 16 to 256");
    if (D < 32 || D > 256 || D % 32)
        return fail(TN_ENOTIMPL, name + ": head_dim " + std::to_string(D) + " is not implemented for a " + format +
                                     " cache; it is a multiple of 32 up to 256");
    // (the attention's grid has up to 8 H workgroups a request in its second dimension)
    if (H < 1 || H > 4096 || P < 0) return fail(TN_EINVAL, name + ": bad cache sizes");
    if (P > INT32_MAX / S) return fail(TN_EVALUE, name + ": a cache holds fewer than 2^31 slots");
    out->pages = (int)P, out->H = (int)H, out->nb = (int)(D / 32);
    out->shift = __builtin_ctzll((unsigned long long)S);
    return TN_OK;
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

tn_status check_planes(const char* op, int pages, const void* a, const void* b, const void* c, const void* d) {
    if (!pages) return TN_OK;  // nothing is read or written
    if (!a || !b || !c || !d) return fail(TN_EVALUE, std::string(op) + ": null cache plane");
    if ((address(a) | address(b) | address(c) | address(d)) & 15)
        return fail(TN_EVALUE, std::string(op) + ": cache planes must be 16-byte aligned");
    return TN_OK;
}

}  // namespace

tn_status paged_check(const char* op, const tn_q4_cache* cache, Pages* out) {
    TN_TRY(check_sizes(op, "q4_0", cache, out));
    out->kc = cache->k_codes, out->kd = cache->k_scales, out->vc = cache->v_codes, out->vd = cache->v_scales;
    return TN_OK;
}

tn_status paged_check(const char* op, const tn_q8_cache* cache, Pages8* out) {
    TN_TRY(check_sizes(op, "q8", cache, out));
    out->kc = cache->k_codes, out->ks = cache->k_scales, out->vc = cache->v_codes, out->vs = cache->v_scales;
    return TN_OK;
}

tn_status paged_check_planes(const char* op, const Pages& c) {
    return check_planes(op, c.pages, c.kc, c.kd, c.vc, c.vd);
}

tn_status paged_check_planes(const char* op, const Pages8& c) {
    return check_planes(op, c.pages, c.kc, c.ks, c.vc, c.vs);
}

namespace {

// ---- pages for requests -------------------------------------------------------

struct PlanArgs {
    const int32_t *fresh, *lens, *state;
    int32_t *lens_out, *table, *free_pages, *state_out, *row_start, *base, *slots, *pos;
    int n, width, shift, pages, tokens;
};

constexpr int PLAN_MAX_N = 4096;

// Inclusive sums over the workgroup's T threads; `red` holds a value per wave and is
// used again only behind the caller's next barrier.
template <int T>
__device__ inline int64_t block_scan(int64_t v, int64_t* red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    if (lane == 63) red[w] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64 - 1; i++) v += i < w ? red[i] : 0;
    return v;
}

// The last index whose value is at most x, of ascending v[0] <= x .. v[n - 1].
__device__ inline int last_at_most(const int32_t* v, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The slot and position of row t: its request by a search of the row starts.
__device__ inline void plan_row(const PlanArgs& a, const int32_t* starts, const int32_t* base, int t) {
    int slot = -1, p = 0;
    if (t < starts[a.n]) {
        const int lo = last_at_most(starts, a.n, t);
        const int b = base[lo];
        if (b >= 0) {
            const int q = b + (t - starts[lo]);
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

// One workgroup: prefix sums over the requests, pages from and to the stack, and the
// rows' slots where they are few (k_plan_rows otherwise). All latency: counts and lengths,
// three sums over the workgroup one after another (rows, pages, what was lacking; four
// where a request has ended, whose counts and lengths are loaded for it first), popped
// pages out to the table and each row's page back from it. 6.5 us for 16 requests of 256
// rows, 13.0 with k_plan_rows for 500 of 60000; a launch is 3.5.
template <int T>
__global__ __launch_bounds__(T) void k_plan(const PlanArgs a, int rows_here) {
    __shared__ int64_t red[2][T / 64];
    __shared__ int32_t s_start[PLAN_MAX_N + 1], s_base[PLAN_MAX_N], s_first[PLAN_MAX_N];
    __shared__ int64_t s_carry[2], s_used[T / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const int size = 1 << a.shift;
    const int64_t most = (int64_t)a.width << a.shift;
    auto held_of = [&](int r) { return min(max((int64_t)a.lens[r], (int64_t)0), most); };
    auto pages_of = [&](int64_t tokens) { return (int)((tokens + size - 1) >> a.shift); };

    // pages of ended requests go back onto the stack
    int64_t count = min(max(a.state[0], 0), a.pages);
    for (int r0 = 0; r0 < a.n; r0 += T) {
        const int r = r0 + tid;
        const bool ended = r < a.n && a.fresh[r] < 0;
        if (!__syncthreads_or(ended)) continue;
        const int give = ended ? pages_of(held_of(r)) : 0;
        const int64_t end = block_scan<T>(give, red[0]);
        if (tid == T - 1) s_carry[0] = end;
        const int64_t at = count + end - give;
        uint64_t givers = __ballot(give > 0);  // a wave a request, its lanes a page each
        while (givers) {
            const int src = __ffsll((unsigned long long)givers) - 1;
            givers &= givers - 1;
            const int g = __shfl(give, src);
            const int64_t to = __shfl(at, src);
            const int64_t row = (int64_t)(r - lane + src) * a.width;
            for (int j = lane; j < g; j += 64)
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
    for (int r0 = 0; r0 < a.n; r0 += T) {
        const int r = r0 + tid;
        int64_t len = 0, add = 0;
        if (r < a.n) {
            const int f = a.fresh[r];
            add = max(f, 0);
            len = f < 0 ? 0 : held_of(r);
        }
        const int held = pages_of(len);
        const int need = (int)min((int64_t)INT32_MAX, ((len + add + size - 1) >> a.shift) - held);
        const int64_t row_end = rows + block_scan<T>(add, red[0]);
        const bool bad = len + add > most || row_end > a.tokens;
        const int want = bad ? 0 : need;
        const int64_t asked = taken + block_scan<T>(want, red[1]);
        const bool ok = !bad && (need == 0 || asked <= count);
        if (tid == T - 1) s_carry[0] = row_end, s_carry[1] = asked;
        if (r < a.n) {
            a.lens_out[r] = (int)(ok ? len + add : len);
            a.base[r] = s_base[r] = ok ? (int)len : -1;
            a.row_start[r + 1] = s_start[r + 1] = (int)min(row_end, (int64_t)a.tokens);
            s_first[r] = (int)min(asked - want, (int64_t)INT32_MAX);
            if (!ok) lacking += max(need, (int)min(add, (int64_t)1));  // its rows or its table may be what ran out
            else if (need) used = asked;
        }
        __syncthreads();
        rows = s_carry[0], taken = s_carry[1];
        __syncthreads();
    }
    // what left the stack: `asked` of the last request that took pages
    const int64_t lack = block_scan<T>(lacking, red[0]);
#pragma unroll
    for (int o = 32; o; o >>= 1) used = max(used, (int64_t)__shfl_xor(used, o));
    if (lane == 0) s_used[tid >> 6] = used;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 64; i++) used = max(used, s_used[i]);
    if (tid == T - 1) {
        a.state_out[0] = (int)(count - used);
        a.state_out[1] = (int)min(lack, (int64_t)INT32_MAX);
    }
    // the pages in the order in which they were asked for: each its request by a search (a
    // request that wants none starts where its successor does, which is found)
    for (int64_t i = tid; i < used; i += T) {
        const int r = last_at_most(s_first, a.n, (int)i);
        a.table[(int64_t)r * a.width + pages_of(s_base[r]) + (i - s_first[r])] = a.free_pages[count - 1 - i];
    }
    if (rows_here) {
        __syncthreads();
        for (int t = tid; t < a.tokens; t += T) plan_row(a, s_start, s_base, t);
    }
}

// The slots of many rows: the row starts in LDS, a row a thread.
__global__ __launch_bounds__(256) void k_plan_rows(const PlanArgs a) {
    __shared__ int32_t s_start[PLAN_MAX_N + 1];
    for (int i = threadIdx.x; i <= a.n; i += 256) s_start[i] = a.row_start[i];
    __syncthreads();
    // (a step past the last of nearly 2^31 rows is no number of 32 bits)
    for (int64_t t = blockIdx.x * 256 + threadIdx.x; t < a.tokens; t += gridDim.x * 256)
        plan_row(a, s_start, a.base, (int)t);
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
    int64_t m;
    bool past;  // read: the output goes past the caches
};

// A workgroup takes ROWS rows of one head, of K or of V. K rows are whole in their plane;
// V rows are bytes of eights of slots. Of a run of eight slots from an aligned one on,
// which a prompt's rows are but for its ends, the bytes leave and come together, 8 a
// lane; other rows' one by one. Bound by memory where rows are many: 8192 bf16 rows of 8
// heads of 128 written in 13.4 us (19 with all bytes one by one), 3.2 TB/s, and read in
// 10.8 (14), 4.0; 65536 read in 56 to 59, 5.8 to 6.1; 16 rows are a launch, 3.7 us.
constexpr int ROWS = 32;

struct Runs {
    int slot[ROWS];   // -1: outside the cache
    int lead[ROWS];   // rows that eight in a row start at, `leads` of them
    int single[ROWS]; // rows in none of these, `singles` of them
    int leads, singles;
};

// The first wave sorts the rows r0 .. of `slots`; all threads wait.
__device__ inline void sort_runs(Runs& s, const int32_t* slots, int64_t r0, int64_t m, const Pages& c) {
    const int t = threadIdx.x;
    if (t < 64) {
        int slot = -1;
        if (t < ROWS && r0 + t < m) {
            slot = slots[r0 + t];
            if (slot < 0 || (slot >> c.shift) >= c.pages) slot = -1;
        }
        // a run starts here: the next seven lanes hold the next seven slots
        const bool first = slot >= 0 && (slot & 7) == 0;
        const int prev = __shfl_up(slot, 1);
        const uint64_t follows = __ballot(t > 0 && slot >= 0 && slot == prev + 1);  // bit t: continues t - 1
        const bool lead = first && t + 8 <= ROWS && ((follows >> (t + 1)) & 0x7f) == 0x7f;
        const uint64_t leads = __ballot(lead);
        uint64_t in = 0;  // lanes of runs
#pragma unroll
        for (int i = 0; i < 8; i++) in |= leads << i;
        const bool alone = t < ROWS && slot >= 0 && !(in >> t & 1);
        const uint64_t singles = __ballot(alone), below = (1ull << t) - 1;
        if (t < ROWS) s.slot[t] = slot;
        if (lead) s.lead[__popcll(leads & below)] = t;
        if (alone) s.single[__popcll(singles & below)] = t;
        if (t == 0) s.leads = __popcll(leads), s.singles = __popcll(singles);
    }
    __syncthreads();
}

// The plane row of a slot and head; the eight that a slot is of.
__device__ inline int64_t plane_row(const Pages& c, int slot, int h) {
    return (((int64_t)(slot >> c.shift) * c.H + h) << c.shift) + (slot & ((1 << c.shift) - 1));
}

template <int DT, int NB>
__global__ __launch_bounds__(256) void k_append(const RowArgs a) {
    __shared__ Runs runs;
    __shared__ uint32_t part[ROWS][4 * NB];  // bytes 4g .. 4g+3 of block b at [g * NB + b]
    __shared__ uint16_t scale[ROWS][NB];
    const int tid = threadIdx.x, h = blockIdx.y;
    const int64_t r0 = (int64_t)blockIdx.x * ROWS;
    sort_runs(runs, a.slots, r0, a.m, a.c);
    const bool v = blockIdx.z;
#pragma unroll
    for (int it = tid; it < ROWS * NB * 4; it += 256) {
        const int g = it & 3, b = (it >> 2) % NB, t = (it >> 2) / NB, slot = runs.slot[t];
        if (slot < 0) continue;  // four lanes together
        uint16_t d;
        const uint32_t w = quantise_part<DT>(v ? a.v : a.k, (r0 + t) * a.stride + (h * NB + b) * 32, g, &d);
        if (v) {
            part[t][g * NB + b] = w;
            if (g == 0) scale[t][b] = d;
        } else {
            const int64_t row = plane_row(a.c, slot, h);
            *reinterpret_cast<uint32_t*>(a.c.kc + row * (16 * NB) + (g * NB + b) * 4) = w;
            if (g == 0) a.c.kd[row * NB + b] = d;
        }
    }
    if (!v) return;
    __syncthreads();
    auto byte = [&](int t, int x) {  // byte column x = c * NB + b
        return part[t][x / NB / 4 * NB + x % NB] >> (x / NB % 4 * 8) & 0xffu;
    };
    for (int it = tid; it < runs.leads * 16 * NB; it += 256) {
        const int t = runs.lead[it / (16 * NB)], x = it % (16 * NB);
        const int64_t row = plane_row(a.c, runs.slot[t], h);  // of the first of the eight
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) w[i >> 2] |= byte(t + i, x) << (8 * (v_place(i) & 3));
        *reinterpret_cast<uint2*>(a.c.vc + row * (16 * NB) + x * 8) = make_uint2(w[0], w[1]);
    }
    for (int it = tid; it < runs.leads * NB * 8; it += 256) {
        const int t = runs.lead[it / (8 * NB)], b = it % (8 * NB) / 8, i = it % 8;
        a.c.vd[plane_row(a.c, runs.slot[t], h) * NB + b * 8 + i] = scale[t + i][b];
    }
    for (int it = tid; it < runs.singles * 16 * NB; it += 256) {
        const int t = runs.single[it / (16 * NB)], x = it % (16 * NB), slot = runs.slot[t];
        const int64_t row = plane_row(a.c, slot & ~7, h);
        a.c.vc[row * (16 * NB) + x * 8 + v_place(slot & 7)] = (uint8_t)byte(t, x);
        if (x < NB) a.c.vd[row * NB + x * 8 + (slot & 7)] = scale[t][x];
    }
}

// PAST: the output goes past the caches.
template <int DT, int NB, bool PAST>
__global__ __launch_bounds__(256) void k_read(const RowArgs a) {
    constexpr int D = 32 * NB, SIZE = DT == TN_F32 ? 4 : 2, PITCH = D * SIZE + 16;
    __shared__ Runs runs;
    __shared__ __align__(16) uint8_t rows[ROWS * PITCH];  // as they leave
    const int tid = threadIdx.x, h = blockIdx.y;
    const int64_t r0 = (int64_t)blockIdx.x * ROWS;
    sort_runs(runs, a.slots, r0, a.m, a.c);
    auto put = [&](int t, int d, float x) {
        if constexpr (DT == TN_F32) *reinterpret_cast<float*>(rows + t * PITCH + d * 4) = x;
        else *reinterpret_cast<uint16_t*>(rows + t * PITCH + d * 2) = DT == TN_BF16 ? bf16_out(x) : f16_out(x);
    };
    auto low = [](uint32_t byte) { return (float)((int)(byte & 15) - 8); };
    if (blockIdx.z == 0) {
#pragma unroll
        for (int it = tid; it < ROWS * NB * 4; it += 256) {
            const int g = it & 3, b = (it >> 2) % NB, t = (it >> 2) / NB, slot = runs.slot[t];
            if (slot < 0) continue;
            const int64_t row = plane_row(a.c, slot, h);
            const uint32_t w = *reinterpret_cast<const uint32_t*>(a.c.kc + row * (16 * NB) + (g * NB + b) * 4);
            const float s = f16_bits_hw(a.c.kd[row * NB + b]);
            float y[2][4];
#pragma unroll
            for (int j = 0; j < 4; j++) y[0][j] = low(w >> (8 * j)) * s, y[1][j] = low(w >> (8 * j + 4)) * s;
            store4<DT>(rows + t * PITCH, 32 * b + 4 * g, y[0]);
            store4<DT>(rows + t * PITCH, 32 * b + 16 + 4 * g, y[1]);
        }
    } else {
        for (int it = tid; it < runs.leads * 16 * NB; it += 256) {
            const int t = runs.lead[it / (16 * NB)], x = it % (16 * NB), b = x % NB, c = x / NB;
            const int64_t row = plane_row(a.c, runs.slot[t], h);
            const uint2 w = *reinterpret_cast<const uint2*>(a.c.vc + row * (16 * NB) + x * 8);
            const uint4 d = *reinterpret_cast<const uint4*>(a.c.vd + row * NB + b * 8);
            const uint32_t ws[2] = {w.x, w.y}, ds[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t byte = ws[i >> 2] >> (8 * (v_place(i) & 3));
                const float s = f16_bits_hw((uint16_t)(ds[i >> 1] >> (16 * (i & 1))));
                put(t + i, 32 * b + c, low(byte) * s);
                put(t + i, 32 * b + 16 + c, low(byte >> 4) * s);
            }
        }
        for (int it = tid; it < runs.singles * 16 * NB; it += 256) {
            const int t = runs.single[it / (16 * NB)], x = it % (16 * NB), b = x % NB, c = x / NB, slot = runs.slot[t];
            const int64_t row = plane_row(a.c, slot & ~7, h);
            const uint32_t byte = a.c.vc[row * (16 * NB) + x * 8 + v_place(slot & 7)];
            const float s = f16_bits_hw(a.c.vd[row * NB + b * 8 + (slot & 7)]);
            put(t, 32 * b + c, low(byte) * s);
            put(t, 32 * b + 16 + c, low(byte >> 4) * s);
        }
    }
    __syncthreads();
    constexpr int PIECES = D * SIZE / 16;
    char* out = static_cast<char*>(blockIdx.z ? a.vo : a.ko);
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(2)));
    constexpr uint32_t NAN2 = DT == TN_F32 ? 0x7fc00000u : DT == TN_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
#pragma unroll
    for (int it = tid; it < ROWS * PIECES; it += 256) {
        const int t = it / PIECES, x = it % PIECES;
        if (r0 + t >= a.m) continue;
        const u4 w = runs.slot[t] < 0 ? (u4){NAN2, NAN2, NAN2, NAN2}
                                      : *reinterpret_cast<const u4*>(rows + t * PITCH + x * 16);
        v4* to = reinterpret_cast<v4*>(out + (((r0 + t) * a.c.H + h) * D) * SIZE + x * 16);
        if constexpr (PAST) __builtin_nontemporal_store((v4)w, to);
        else *to = w;
    }
}

template <int DT>
void rows_launch(hipStream_t st, const RowArgs& a, bool append) {
    const dim3 grid((unsigned)cdiv(a.m, ROWS), (unsigned)a.c.H, 2);
#define TN_ROWS(NB)                                                                    \
    case NB:                                                                           \
        if (append) hipLaunchKernelGGL((k_append<DT, NB>), grid, dim3(256), 0, st, a); \
        else if (a.past) hipLaunchKernelGGL((k_read<DT, NB, true>), grid, dim3(256), 0, st, a); \
        else hipLaunchKernelGGL((k_read<DT, NB, false>), grid, dim3(256), 0, st, a);   \
        break;
    switch (a.c.nb) {
        TN_ROWS(1) TN_ROWS(2) TN_ROWS(3) TN_ROWS(4) TN_ROWS(5) TN_ROWS(6) TN_ROWS(7) TN_ROWS(8)
    }
#undef TN_ROWS
}

tn_status rows_at(hipStream_t st, int dtype, const RowArgs& a, bool append) {
    if (dtype == TN_F32) rows_launch<TN_F32>(st, a, append);
    else if (dtype == TN_BF16) rows_launch<TN_BF16>(st, a, append);
    else rows_launch<TN_F16>(st, a, append);
    TN_LAUNCHED();
    return TN_OK;
}

tn_status row_check(const char* op, const tn_q4_cache* cache, int dtype, int64_t m, RowArgs* a) {
    TN_TRY(paged_check(op, cache, &a->c));
    if (dtype != TN_F32 && dtype != TN_BF16 && dtype != TN_F16)
        return fail(TN_ENOTIMPL, std::string(op) + ": rows must be float32, bfloat16 or float16");
    if (m < 0) return fail(TN_EINVAL, std::string(op) + ": bad sizes");
    a->m = m;
    // 8 threads a row, a grid of fewer than 2^32
    if (m > 1 << 28) return fail(TN_EVALUE, std::string(op) + ": shape too large");
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
    // rows in the workgroup that plans, or in a launch of their own (us: 256 requests, 4096
    // rows, 11.5 and 11.8; 100 of 8192, 14.5 and 10.9; 16 of 16, 6.6 and 7.9)
    const bool here = tokens <= 4096;
    // 256 threads, or 1024 and their longer barriers (16 requests, 6.6 and 10.5; 256 of 1024
    // rows, 7.5 and 8.9; of 4096, 17.6 and 11.5; 500 requests, 18.1 and 15.4; 100 with rows of
    // their own launch, 8.8 and 10.9)
    const bool small = n <= 256 && (tokens <= 1024 || !here);
    hipStream_t st = (hipStream_t)stream;
    if (small) hipLaunchKernelGGL(k_plan<256>, dim3(1), dim3(256), 0, st, a, (int)here);
    else hipLaunchKernelGGL(k_plan<1024>, dim3(1), dim3(1024), 0, st, a, (int)here);
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
    return rows_at((hipStream_t)stream, dtype, a, true);
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
    // Outputs that the L2 caches hold between them stay in them for the kernel that reads them
    // next; larger ones go past. (us, through the caches and past them, rows of 8 heads of 128,
    // bf16, ten outputs in turn. Alone: 4096 rows, 16 MB, 7.2 and 5.9; 8192 rows, exactly at
    // the limit and so through, 14.4 and 9.6; 9000, 15.8 and 10.3; 65536, 90 and 56. The
    // caches' share is written back at a later kernel's cost: with one that reads the output
    // right after, 4096 rows 12.2 and 11.9, 6000 17.1 and 18.5, 8192 22.7 and 23.0, 9000 24.9
    // and 25.8, 32768 75 and 74.)
    a.past = 2 * m * a.c.H * a.c.nb * 32 * (dtype == TN_F32 ? 4 : 2) > (32 << 20);
    return rows_at((hipStream_t)stream, dtype, a, false);
}

}  // extern "C"
