// paged_cache.hip -- the tables of a paged cache built on the device from
// request lengths, rows of keys and values quantized into its pages, and read
// back.
#include "paged.hpp"

namespace lamd {

// ---- tables -----------------------------------------------------------------

__global__ void page_reset_kernel(PageTables t) {
    const long n = (long)t.requests * t.max_pages;
    const long i0 = (long)blockIdx.x * blockDim.x + threadIdx.x, step = (long)gridDim.x * blockDim.x;
    for (long i = i0; i < n; i += step) t.table[i] = -1;
    for (long i = i0; i < t.requests; i += step) t.held[i] = 0;
    for (long i = i0; i < t.pages; i += step) t.free_pages[i] = t.pages - 1 - (int)i;
    if (i0 == 0) *t.free_count = t.pages;
}

hipError_t launch_page_reset(const PageTables& t, hipStream_t s) {
    const long n = (long)t.requests * t.max_pages > t.pages ? (long)t.requests * t.max_pages : t.pages;
    const long blocks = (n + 255) / 256;
    hipLaunchKernelGGL(page_reset_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, s, t);
    return hipGetLastError();
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// One workgroup also fills the rows up to these counts (its row starts in LDS).
constexpr int kFoldRequests = 4096;
constexpr int kFoldRows = 4096;

// Inclusive sum over the workgroup in thread order; every thread gets the total.
__device__ __forceinline__ long long block_scan(long long v, long long* wave_sum, long long* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    __syncthreads();  // wave_sum of the previous call has been read
    if (lane == 63) wave_sum[wave] = v;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
        const long long x = wave_sum[w];
        if (w < wave) before += x;
        all += x;
    }
    *total = all;
    return v + before;
}

// The rows of a step, request by request: row_start is the running sum of the
// new tokens (held to `rows`), and a request takes ceil((len + new) / page) -
// held pages off the top of the free stack, in request order, so the page ids
// depend on nothing but the lengths.  A request takes part whole or not at
// all: one whose pages, row or table space run out keeps its length, and its
// rows get position and slot -1.  One workgroup, because the running sums are
// serial: what it costs is the latency of its few dependent steps (7.2 us for
// the 64 requests of a decode step).  FILL also writes the pages and rows; otherwise
// page_fill_kernel does, one workgroup a request, from scratch {first
// position or -1, pages taken, top of the stack at its first page, pages held
// before}.
template <bool FILL>
__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(PageTables t, const int32_t* __restrict__ lens,
                                                                 const int32_t* __restrict__ new_tokens, int rows,
                                                                 PlanOut o) {
    __shared__ long long sum_rows[kPlanWaves], sum_pages[kPlanWaves];
    __shared__ int start_s[FILL ? kFoldRequests + 1 : 1];
    __shared__ int base_s[FILL ? kFoldRequests : 1];
    __shared__ int taken_s;
    const int tid = threadIdx.x;
    const long long free0 = min(max(*t.free_count, 0), t.pages);  // (a table that was never reset stays in bounds)
    const long long room = (long long)t.max_pages * t.page;
    long long rows_before = 0, pages_before = 0;
    if (tid == 0) {
        taken_s = 0;
        o.row_start[0] = 0;
        if (FILL) start_s[0] = 0;
    }
    for (int r0 = 0; r0 < t.requests; r0 += kPlanThreads) {
        const int r = r0 + tid;
        const bool in = r < t.requests;
        long long base = 0, n = 0;
        int held = 0;
        if (in) {
            base = lens[r] > 0 ? lens[r] : 0;
            n = new_tokens[r] > 0 ? new_tokens[r] : 0;
            held = min(max(t.held[r], 0), t.max_pages);
        }
        long long total;
        const long long row_end = block_scan(n, sum_rows, &total) + rows_before;
        rows_before += total;
        bool ok = base + n <= room && row_end <= rows;
        long long want = 0;
        if (ok && in) {
            want = (base + n + t.page - 1) / t.page - held;
            if (want < 0) want = 0;
        }
        const long long page_end = block_scan(want, sum_pages, &total) + pages_before;
        pages_before += total;
        ok = ok && (want == 0 || page_end <= free0);
        if (!ok) want = 0;
        if (in) {
            const int end = (int)(row_end < rows ? row_end : rows);
            const int top = (int)(free0 - 1 - (page_end - want));
            o.row_start[r + 1] = end;
            o.lens[r] = (int32_t)(ok ? base + n : base);
            if (FILL) {
                start_s[r + 1] = end;
                base_s[r] = ok ? (int)base : -1;
                t.held[r] = held + (int)want;
            } else {
                int4 sc = make_int4(ok ? (int)base : -1, (int)want, top, held);
                ((int4*)o.scratch)[r] = sc;
            }
            if (want > 0) atomicMax(&taken_s, (int)page_end);
            if (FILL && want <= 16) {
                for (int j = 0; j < (int)want; ++j) t.table[(long)r * t.max_pages + held + j] = t.free_pages[top - j];
            }
        }
        if (FILL) {  // requests of many pages: a wave each
            unsigned long long many = __ballot(in && want > 16);
            while (many) {
                const int l = __builtin_ctzll(many);
                many &= many - 1;
                const int w = __shfl((int)want, l, 64), h = __shfl(held, l, 64);
                const int top = __shfl((int)(free0 - 1 - (page_end - want)), l, 64);
                const long at = (long)(r0 + (tid & ~63) + l) * t.max_pages + h;
                for (int j = tid & 63; j < w; j += 64) t.table[at + j] = t.free_pages[top - j];
            }
        }
    }
    __syncthreads();
    if (tid == 0) *t.free_count = (int32_t)(free0 - taken_s);
    if (FILL) {
        for (int row = tid; row < rows; row += kPlanThreads) {
            // the request whose rows hold this one: the last start at or before it
            int lo = 0, hi = t.requests + 1;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start_s[mid] <= row) lo = mid;
                else hi = mid;
            }
            int req = -1, pos = -1, slot = -1;
            if (lo < t.requests) {
                req = lo;
                if (base_s[lo] >= 0) {
                    pos = base_s[lo] + row - start_s[lo];
                    slot = t.table[(long)lo * t.max_pages + pos / t.page] * t.page + pos % t.page;
                }
            }
            o.request[row] = req;
            o.positions[row] = pos;
            o.slots[row] = slot;
        }
    }
}

// Pages and rows of request blockIdx.x (the last block: rows behind the last
// request), from page_plan_kernel's scratch.
__global__ __launch_bounds__(256) void page_fill_kernel(PageTables t, int rows, PlanOut o) {
    const int r = blockIdx.x;
    const int first = threadIdx.x + blockIdx.y * blockDim.x, step = blockDim.x * gridDim.y;
    if (r == t.requests) {
        for (long row = (long)o.row_start[r] + first; row < rows; row += step) {
            o.request[row] = o.positions[row] = o.slots[row] = -1;
        }
        return;
    }
    const int4 sc = ((const int4*)o.scratch)[r];
    const int base = sc.x, want = sc.y, top = sc.z, held = sc.w;
    int32_t* table = t.table + (long)r * t.max_pages;
    for (int j = first; j < want; j += step) table[held + j] = t.free_pages[top - j];
    if (want > 0 && first == 0) t.held[r] = held + want;
    const int start = o.row_start[r], end = o.row_start[r + 1];
    for (int row = start + first; row < end; row += step) {
        int pos = -1, slot = -1;
        if (base >= 0) {
            pos = base + row - start;
            const int i = pos / t.page;
            slot = (i < held ? table[i] : t.free_pages[top - (i - held)]) * t.page + pos % t.page;
        }
        o.request[row] = r;
        o.positions[row] = pos;
        o.slots[row] = slot;
    }
}

hipError_t launch_page_plan(const PageTables& t, const int32_t* lens, const int32_t* new_tokens, int rows,
                            const PlanOut& o, hipStream_t s) {
    if (t.requests <= kFoldRequests && rows <= kFoldRows) {
        hipLaunchKernelGGL(page_plan_kernel<true>, dim3(1), dim3(kPlanThreads), 0, s, t, lens, new_tokens, rows, o);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(page_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, s, t, lens, new_tokens, rows, o);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // long requests spread over several workgroups
    int parts = rows / (1024 * (t.requests < 64 ? t.requests : 64));
    parts = parts < 1 ? 1 : (parts > 64 ? 64 : parts);
    hipLaunchKernelGGL(page_fill_kernel, dim3((unsigned)t.requests + 1, parts), dim3(256), 0, s, t, rows, o);
    return hipGetLastError();
}

// Pages of the requests marked done go back on the stack, in request order.
__global__ __launch_bounds__(kPlanThreads) void page_release_kernel(PageTables t, const uint8_t* __restrict__ done) {
    __shared__ long long sum[kPlanWaves];
    const int tid = threadIdx.x;
    const int free0 = min(max(*t.free_count, 0), t.pages);
    long long before = 0;
    for (int r0 = 0; r0 < t.requests; r0 += kPlanThreads) {
        const int r = r0 + tid;
        int n = 0;
        if (r < t.requests && done[r]) {
            n = t.held[r];
            if (n > t.max_pages) n = t.max_pages;
        }
        long long total;
        const long long at = block_scan(n, sum, &total) + before - n;
        before += total;
        if (n > 0) t.held[r] = 0;
        unsigned long long some = __ballot(n > 0);
        while (some) {
            const int l = __builtin_ctzll(some);
            some &= some - 1;
            const int cnt = __shfl(n, l, 64);
            const long long to = free0 + __shfl(at, l, 64);
            int32_t* row = t.table + (long)(r0 + (tid & ~63) + l) * t.max_pages;
            for (int j = tid & 63; j < cnt; j += 64) {
                if (to + j < t.pages) t.free_pages[to + j] = row[j];
                row[j] = -1;
            }
        }
    }
    __syncthreads();
    if (tid == 0) *t.free_count = (int32_t)(free0 + before < t.pages ? free0 + before : t.pages);
}

hipError_t launch_page_release(const PageTables& t, const uint8_t* done, hipStream_t s) {
    hipLaunchKernelGGL(page_release_kernel, dim3(1), dim3(kPlanThreads), 0, s, t, done);
    return hipGetLastError();
}

// ---- append and read ------------------------------------------------------------

constexpr float kMaxFinite = 3.402823466e38f;
constexpr float kTinyAmax = 0x1p-100f;  // below it a block's values are zeros: its scale keeps full precision

template <typename T>
__device__ __forceinline__ float as_f32(T v);
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_f32<uint16_t>(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= kMaxFinite ? a : 0.0f;  // NaN and infinities have no part in the scale
}

// round-half-away(x / s) of four finite values with |x / s| <= 127 (and a
// rounding), exactly: the estimate is at most one off, and the sign of
// |x| - (c +- 1/2) s, one fused operation, is exact (s >= 2^-107).  s is
// infinite and inv 0 for a block of zeros.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float s, float inv) {
    const float x[4] = {a, b, c, d};
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float q = x[j] * inv, m = fabsf(x[j]);
        float h = truncf(fabsf(q) + 0.5f);
        const float below = __builtin_fmaf(0.5f - h, s, m), above = __builtin_fmaf(-0.5f - h, s, m);
        h += below < 0.0f ? -1.0f : (above >= 0.0f ? 1.0f : 0.0f);
        w = __builtin_amdgcn_cvt_pk_u8_f32(copysignf(h, x[j]) + 128.0f, j, w);
    }
    return w ^ 0x80808080u;
}

// Four codes of scale `from` at the larger scale `to`: round-half-away(c from /
// to), exactly.  c from and (h +- 1/2) to are exact in fp64, so the estimate
// (inv = 1 / to) needs no more than a comparison on either side.
__device__ __forceinline__ uint32_t recode4(uint32_t w, double from, double to, double inv) {
    uint32_t z = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int c = (int8_t)(w >> (8 * b));
        const double p = (double)abs(c) * from;
        double h = floor(p * inv + 0.5);
        if (p < (h - 0.5) * to) h -= 1.0;
        else if (p >= (h + 0.5) * to) h += 1.0;
        const int i = (int)h;
        z |= (uint32_t)(uint8_t)(c < 0 ? -i : i) << (8 * b);
    }
    return z;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

// Four consecutive elements (vec: one load).
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float* x) {
    if (vec) {
        if (sizeof(T) == 4) {
            const float4 f = *(const float4*)p;
            x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
        } else {
            const uint2 u = *(const uint2*)p;
            x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xffff0000u);
            x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = as_f32<T>(p[i]);
    }
}

constexpr int kWindow = 16;  // rows whose runs one workgroup looks for

// One side of one head of a run of n tokens from offset `off` of a page: its
// scale (at *scale_at), then its codes.  src is the run's first row.
//
// Keys: unit u is dimensions 4 (u % D4) .. of token u / D4, one word of codes.
// Values: unit u is the same of four tokens, quad by quad, four words.  2048
// values of a run stay in registers between the search for the largest and the
// rounding; longer runs are read again.
template <typename T, int HD, bool V>
__device__ __forceinline__ void append_run(const T* src, long stride, int off, int n, int8_t* codes, float* scale_at,
                                           bool vec, int lane) {
    constexpr int D4 = HD / 4;
    constexpr int PER = V ? 2 : 8;  // units of a lane in registers
    const float had = off == 0 ? 0.0f : *scale_at;
    const int q0 = off >> 2;
    const int units = V ? (((off + n + 3) >> 2) - q0) * D4 : n * D4;
    float x[8][4];
    auto fetch = [&](int u0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int u = u0 + lane + 64 * i;
            const int t = V ? 4 * (q0 + u / D4) - off : u / D4;
            const T* p = src + (long)t * stride + 4 * (u % D4);
#pragma unroll
            for (int j = 0; j < 8 / PER; ++j) {
                float* y = x[V ? 4 * i + j : i];
                if (u < units && (!V || (t + j >= 0 && t + j < n))) load4<T>(p + j * stride, vec, y);
                else y[0] = y[1] = y[2] = y[3] = 0.0f;
            }
        }
    };
    float big = 0.0f;
    float zero = 0.0f;  // becomes NaN with a value that is not finite
#pragma unroll 1
    for (int u0 = 0; u0 < units; u0 += 64 * PER) {
        fetch(u0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                big = fmaxf(big, fabsf(x[i][j]));
                zero = __builtin_fmaf(x[i][j], 0.0f, zero);
            }
        }
    }
    const bool odd = __any(zero != 0.0f);  // (NaN)
    if (odd) {
        big = 0.0f;
#pragma unroll 1
        for (int u0 = 0; u0 < units; u0 += 64 * PER) {
            fetch(u0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) big = fmaxf(big, finite_abs(x[i][j]));
            }
        }
    }
    big = wave_max(big);
    const float own = big < kTinyAmax ? 0.0f : big / 127.0f;
    const float to = fmaxf(had, own);
    const float inv = to > 0.0f ? 1.0f / to : 0.0f, div = to > 0.0f ? to : __builtin_inff();
    const bool grows = off > 0 && to > had;
    const double wide_inv = grows ? 1.0 / (double)to : 0.0;
    if (grows) {
        // earlier tokens (values: whole words; one shared with the run is done below)
        const int words = V ? q0 * HD : off * D4;
        for (int i0 = lane; i0 < words; i0 += 64 * 4) {
            uint32_t* at[4];
            uint32_t y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + 64 * k;
                at[k] = (uint32_t*)(codes + (V ? v_offset(4 * (i / HD), i % HD, HD) : k_offset(i / D4, 4 * (i % D4), HD)));
                y[k] = i < words ? *at[k] : 0u;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i0 + 64 * k < words) *at[k] = recode4(y[k], had, to, wide_inv);
            }
        }
    }
#pragma unroll 1
    for (int u0 = 0; u0 < units; u0 += 64 * PER) {
        if (units > 64 * PER) fetch(u0);
        if (odd) {
            // NaN is stored as 0, an infinity as the largest code
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y = x[i][j];
                    x[i][j] = y != y ? 0.0f : copysignf(fminf(fabsf(y), fminf(127.0f * to, kMaxFinite)), y);
                }
            }
        }
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // values: word i is dimension i % 4 of unit i / 4, its bytes the tokens
            const int r = V ? i & 4 : i, j = i & 3;
            w[i] = V ? codes4(x[r][j], x[r + (V ? 1 : 0)][j], x[r + (V ? 2 : 0)][j], x[r + (V ? 3 : 0)][j], div, inv)
                     : codes4(x[r][0], x[r][1], x[r][2], x[r][3], div, inv);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int u = u0 + lane + 64 * i;
            if (u >= units) continue;
            if (!V) {
                *(uint32_t*)(codes + k_offset(off + u / D4, 4 * (u % D4), HD)) = w[i];
                continue;
            }
            const int q = q0 + u / D4;
            const int t0 = 4 * q - off;  // its first token in the run
            uint32_t mask = 0xffffffffu;
            if (t0 < 0) mask <<= -8 * t0;
            if (t0 + 4 > n) mask &= 0xffffffffu >> (8 * (t0 + 4 - n));
            uint32_t* at = (uint32_t*)(codes + v_offset(4 * q, 4 * (u % D4), HD));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t z = w[(4 * i + j) & 7];
                if (mask != 0xffffffffu) {
                    uint32_t old = at[4 * j];
                    if (grows && t0 < 0) old = recode4(old, had, to, wide_inv);
                    z = (z & mask) | (old & ~mask);
                }
                at[4 * j] = z;
            }
        }
    }
    if (lane == 0) *scale_at = to;
}

// Jobs are (run, head, side), a wave each.  A run is the consecutive rows
// whose slots follow one another within one page, and belongs to the window
// of its first row.  The page's scale is the larger of what it had (unless the
// run starts the page: then nothing of it counts any more) and the run's
// largest magnitude / 127.  When it grows, the codes of the earlier tokens are
// rounded again at the new scale.  13.8 k rows of 5 heads of 128, bf16, pages of
// 32: 48 us (53 MB), bound by each wave's chain of loads, maximum, second read
// and stores; at most 168 registers, for three waves a SIMD (two, or four with
// spills: a tenth more).
template <typename T, int HD>
__global__ __launch_bounds__(256, 3) void kv_append_kernel(KvPages c, const T* __restrict__ k, const T* __restrict__ v,
                                                        int rows, long k_stride, long v_stride, bool vec,
                                                        const int32_t* __restrict__ slots) {
    const int lane = threadIdx.x & 63;
    const int row0 = blockIdx.x * kWindow;
    // rows of the window that start a run
    bool leads = false;
    if (lane < kWindow && row0 + lane < rows) {
        const int row = row0 + lane, slot = slots[row];
        leads = slot >= 0 && slot < c.pages * c.page && !(row > 0 && slot % c.page > 0 && slots[row - 1] == slot - 1);
    }
    unsigned long long left = __ballot(leads);
    const int sides = 2 * c.kv_heads, waves = gridDim.y * 4;
    int job = blockIdx.y * 4 + (threadIdx.x >> 6);
    for (; left; left &= left - 1, job -= sides) {
        if (job >= sides) continue;  // (of a later run)
        const int row = row0 + __builtin_ctzll(left);
        const int slot = slots[row];
        const int page = slot / c.page, off = slot % c.page;
        int n = 0;  // tokens of the run
        for (int base = 0; base < c.page; base += 64) {
            const int t = base + lane;
            const bool more = row + t < rows && off + t < c.page && slots[row + t] == slot + t;
            const unsigned long long m = ~__ballot(more);
            if (m) {
                n = base + __builtin_ctzll(m);
                break;
            }
            n = base + 64;
        }
        for (; job < sides; job += waves) {
            const int head = job >> 1;
            const long at = (long)page * c.kv_heads + head, block = at * (c.page * HD);
            if (job & 1) {
                append_run<T, HD, true>(v + (long)row * v_stride + head * HD, v_stride, off, n, c.v + block, c.v_scale + at,
                                        vec, lane);
            } else {
                append_run<T, HD, false>(k + (long)row * k_stride + head * HD, k_stride, off, n, c.k + block,
                                         c.k_scale + at, vec, lane);
            }
        }
    }
}

template <typename T>
static hipError_t append_typed(const KvPages& c, const void* k, const void* v, int rows, long ks, long vs,
                               const int32_t* slots, hipStream_t s) {
    const uintptr_t m = 4 * sizeof(T) - 1;
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & m) == 0 && ((ks | vs) & 3) == 0;
    // few rows: a wave for every job there may be; many: runs of several rows
    // are likely, and waves go on to further runs where there are more
    const int jobs = 2 * c.kv_heads * (rows < 1024 ? (rows < kWindow ? rows : kWindow) : 1);
    const dim3 grid((unsigned)ceil_div(rows, kWindow), (unsigned)(jobs < 4 * 65535 ? ceil_div(jobs, 4) : 65535));
#define APPEND(HD)                                                                                               \
    case HD:                                                                                                     \
        hipLaunchKernelGGL((kv_append_kernel<T, HD>), grid, dim3(256), 0, s, c, (const T*)k, (const T*)v, rows, ks, \
                           vs, vec, slots);                                                                      \
        break;
    switch (c.hd) {
        APPEND(32)
        APPEND(64)
        APPEND(128)
        APPEND(256)
        default: return hipErrorInvalidValue;
    }
#undef APPEND
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvPages& c, const void* k, const void* v, int type, int rows, long k_stride,
                            long v_stride, const int32_t* slots, hipStream_t s) {
    return type == ROW_BF16 ? append_typed<uint16_t>(c, k, v, rows, k_stride, v_stride, slots, s)
                            : append_typed<float>(c, k, v, rows, k_stride, v_stride, slots, s);
}

// Values code * scale of given slots; no slot reads as zeros.  A workgroup
// takes 16 rows of one head: the codes of values, whose tokens lie side by
// side, are read with the rows on neighbouring lanes (rows of one page share
// their lines) and turned in LDS, so that both sides are written in whole lines.
__global__ __launch_bounds__(256) void kv_read_kernel(KvPages c, const int32_t* __restrict__ slots, int rows,
                                                      float* __restrict__ k, float* __restrict__ v) {
    __shared__ int8_t turn[256 * 17];
    const int row0 = blockIdx.x * 16, h = blockIdx.y;
    const int t = threadIdx.x;
    {
        const int row = row0 + (t & 15);
        const int slot = row < rows ? slots[row] : -1;
        const bool in = slot >= 0 && slot < c.pages * c.page;
        const int page = in ? slot / c.page : 0, off = in ? slot % c.page : 0;
        const int8_t* src = c.v + ((long)page * c.kv_heads + h) * ((long)c.page * c.hd) + v_offset(off, 0, c.hd);
#pragma unroll 4
        for (int d = t >> 4; d < c.hd; d += 16) turn[d * 17 + (t & 15)] = in ? src[16 * d] : (int8_t)0;
    }
    __syncthreads();
    const int d4 = c.hd >> 2;
    for (int i = t; i < 16 * d4; i += 256) {
        const int rr = i / d4, d = 4 * (i % d4), row = row0 + rr;
        if (row >= rows) break;
        const int slot = slots[row];
        const bool in = slot >= 0 && slot < c.pages * c.page;
        const int page = in ? slot / c.page : 0, off = in ? slot % c.page : 0;
        const long ph = (long)page * c.kv_heads + h;
        const float fk = in ? c.k_scale[ph] : 0.0f, fv = in ? c.v_scale[ph] : 0.0f;
        uint32_t w = 0;
        if (in) w = *(const uint32_t*)(c.k + ph * ((long)c.page * c.hd) + k_offset(off, d, c.hd));
        const long at = ((long)row * c.kv_heads + h) * c.hd + d;
        float a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = in ? (float)(int8_t)(w >> (8 * j)) * fk : 0.0f;
            b[j] = in ? (float)turn[(d + j) * 17 + rr] * fv : 0.0f;
        }
        *(float4*)(k + at) = make_float4(a[0], a[1], a[2], a[3]);
        *(float4*)(v + at) = make_float4(b[0], b[1], b[2], b[3]);
    }
}

hipError_t launch_kv_read(const KvPages& c, const int32_t* slots, int rows, float* k, float* v, hipStream_t s) {
    hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)ceil_div(rows, 16), (unsigned)c.kv_heads), dim3(256), 0, s, c, slots,
                       rows, k, v);
    return hipGetLastError();
}

}  // namespace lamd
