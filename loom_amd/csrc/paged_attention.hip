// paged_attention.hip -- causal attention of new rows over a paged cache of
// int8 codes (paged.hpp): one kernel for single decode rows, chunks of a
// prompt, and both in one call.
//
//   out[row, h] = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q.k_t - max)
// over t <= position(row), with k_t = kc_t ks, v_t = vc_t vs of t's page.
//
// The matrix cores read the keys' codes as they are stored: q is written in
// fixed point as three signed 8-bit digits (23 bits and sign) of its largest
// magnitude, and v_mfma_i32_16x16x64_i8 forms every digit's dot product exactly
// in 32 bits; the digits' sums are joined in fp32.  That is no more error than
// an fp32 product has.  (Two digits would do for bf16 rows without outliers;
// they saved nothing on decode rows and 4 % on chunks.)
// The values' codes become fp16 (exact) and meet p as one fp16 factor (bf16
// rows) or as the sum of two (22 bits, fp32 rows).
//
// A wave owns 16 columns: (row, head of the group) pairs of one request and
// key/value head.  It computes scores transposed, S^T = K Q^T, so lane (n, g)
// (n = lane & 15, g = lane >> 4) holds column n's scores of the 16 tokens
// 16g .. 16g+15 of a 64-token step: row r of the K operand of tile t is token
// 16 (r >> 2) + 4 t + (r & 3).  That is the B operand of O^T = V^T P^T as it
// stands, so probabilities never leave registers, nothing but the final join
// uses LDS, and a lane's 16 tokens lie in one page: its scales are one factor.
#include "paged.hpp"

namespace lamd {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;         // tokens of one step
constexpr int QD = 3;             // digits of q
constexpr int kMaxSplits = 64;    // parts of one context (a wave joins them, a lane each)
// fp16 value of a probability of 1, and how far (log2) a score may pass the
// maximum that the sums are relative to before they are rescaled: 2^(9 + 6)
// stays in fp16's range, and few steps rescale
constexpr float kPeak = 512.0f;
constexpr float kSlack = 6.0f;
constexpr float kHuge = 0x1p22f;  // scores from which the fused difference to the maximum is too coarse
constexpr float kNegInf = -__builtin_inff();

struct AttnParams {
    const int8_t* k;
    const int8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* table;
    const int32_t* row_start;
    const int32_t* positions;
    const void* q;
    void* out;
    float* part_o;    // [split][row][head][hd]
    float* part_ml;   // [split][row][head][2]
    int32_t* active;  // [row][head]: parts of this row's context
    int pages, shift, kv_heads, max_pages, requests, rows, heads, group, splits, type, max_context;
    int min_steps;       // steps of a part
    int hi_cols;  // requests of up to so many columns go to the rows kernel, others to the chunk kernel
    long q_stride, out_stride;
    float scale2;  // scale * log2(e)
    bool vec;      // rows of q and out are 16-byte aligned
};

// Largest over the four lanes that share a column (lanes n + 16 g): the
// exchange instructions swap rows of 16 and halves in registers.
__device__ __forceinline__ float column_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float column_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float shfl_xor_f(float v, int m) { return __shfl_xor(v, m, 64); }

__device__ __forceinline__ float bf16_f(uint32_t hi16) { return __uint_as_float(hi16 << 16); }

__device__ __forceinline__ uint32_t f_bf16(float f) {  // round to nearest, ties to even; NaN stays NaN
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// 16 consecutive elements of a row as fp32.
__device__ __forceinline__ void load16(const void* base, int type, long at, bool vec, float* x) {
    if (type == ROW_BF16) {
        const uint16_t* p = (const uint16_t*)base + at;
        if (vec) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 u = ((const uint4*)p)[i];
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[8 * i + 2 * j] = bf16_f(w[j] & 0xffffu);
                    x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = bf16_f(p[i]);
        }
    } else if (type == ROW_F32) {
        const float* p = (const float*)base + at;
        if (vec) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 f = ((const float4*)p)[i];
                x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = p[i];
        }
    } else {
        const double* p = (const double*)base + at;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = (float)p[i];
    }
}

// 4 consecutive elements of an output row.
__device__ __forceinline__ void store4(void* base, int type, long at, bool vec, const float* x) {
    if (type == ROW_BF16) {
        uint16_t* p = (uint16_t*)base + at;
        if (vec) {
            *(uint2*)p = make_uint2(f_bf16(x[0]) | (f_bf16(x[1]) << 16), f_bf16(x[2]) | (f_bf16(x[3]) << 16));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = (uint16_t)f_bf16(x[i]);
        }
    } else if (type == ROW_F32) {
        float* p = (float*)base + at;
        if (vec) {
            *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = x[i];
        }
    } else {
        double* p = (double*)base + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = (double)x[i];
    }
}

// Column tiles of `ct` columns: request r has the launch's tiles from
// start_r * group / ct + r on (the sum of the earlier requests' rounded-up
// tile counts is never more), so a tile finds its request by one search and no
// list of tiles has to be built.  Returns the request or -1; a wave searches
// 64 requests at a time.
__device__ __forceinline__ int find_request(const AttnParams& a, int ct, int x, int lane, int* first_tile) {
    int lo = 0, hi = a.requests;
    while (true) {
        const int step = (hi - lo + 63) >> 6;
        const int r = lo + lane * step;
        long f = 0;
        if (r < hi) {
            int s = a.row_start[r];
            s = s < 0 ? 0 : (s > a.rows ? a.rows : s);
            f = (long)s * a.group / ct + r;
        }
        const unsigned long long at_or_before = __ballot(r < hi && f <= x);
        if (!at_or_before) return -1;
        const int last = 63 - __builtin_clzll(at_or_before);
        lo += last * step;
        if (step == 1) {
            *first_tile = __shfl((int)f, last, 64);
            return lo;
        }
        hi = lo + step < hi ? lo + step : hi;
    }
}

// 16 columns of one wave.
template <int HD, int PL>
struct Wave {
    static constexpr int NS = HD >= 64 ? HD / 64 : 1;  // 64-dimension steps of the score product
    static constexpr int ND = HD / 16;                 // 16-dimension tiles of the output
    v4i qd[QD][NS];
    float qf;  // value of one unit of q's fixed point, with scale * log2(e)
    v4f o[ND];
    // maximum that the sums are relative to (base: 0 for none yet), sum, largest
    // scale of values, fp16 value of a probability of 1 at a scale of 1
    float m, base, l, ref, unit;

    // q's digits of this lane: column n's dimensions 64 s + 16 g ..
    __device__ __forceinline__ void load_q(const AttnParams& a, long at, bool valid, int g) {
        float x[NS][16];
        float big = 0.0f;
        bool bad = false;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (valid && 64 * s + 16 * g < HD) {
                load16(a.q, a.type, at + 64 * s + 16 * g, a.vec, x[s]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[s][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                bad = bad || !(fabsf(x[s][i]) <= 3.402823466e38f);
                big = fmaxf(big, fabsf(x[s][i]));
            }
        }
        big = column_max(big);
        const float nan = column_sum(bad ? __builtin_nanf("") : 0.0f);
        // largest fixed-point value: just under the digits' own, 127 * (1 + 256 + 65536)
        constexpr float kTop = 8355000.0f;
        const bool zero = big < 0x1p-100f;
        const float inv = zero ? 0.0f : (a.scale2 < 0.0f ? -kTop : kTop) / big;
        qf = (zero ? 0.0f : big / kTop) * fabsf(a.scale2);
        l += nan;  // a query that is not finite: NaN to the end
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float f = rintf(x[s][4 * w + i] * inv);
                    f = fminf(fmaxf(f, -kTop), kTop);  // (NaN, infinities: any digits, the sum is NaN)
                    y[i] = ((uint32_t)(int)f + 0x80808080u) ^ 0x80808080u;  // signed digits, lowest byte first
                }
                const uint32_t a01 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u);
                const uint32_t a23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
                qd[0][s][w] = (int)__builtin_amdgcn_perm(a23, a01, 0x05040100u);
                qd[1][s][w] = (int)__builtin_amdgcn_perm(a23, a01, 0x07060302u);
                const uint32_t b01 = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602u);
                const uint32_t b23 = __builtin_amdgcn_perm(y[3], y[2], 0x0c0c0602u);
                qd[2][s][w] = (int)__builtin_amdgcn_perm(b23, b01, 0x05040100u);
            }
        }
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        m = kNegInf;
        base = 0.0f;
        l = 0.0f;
        ref = 0x1p-100f;  // under every scale that holds a value
        unit = kPeak / ref;
    }

    // Scores of tile t (digits joined, without their scale): keys in rows.
    __device__ __forceinline__ void tile(const v4i* k, float* x) const {
        v4i acc[QD];
#pragma unroll
        for (int d = 0; d < QD; ++d) acc[d] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int d = 0; d < QD; ++d) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[s], qd[d][s], acc[d], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (a digit's sum is at most 2^22 at head_dim 256: 256 times that fits)
            x[i] = __builtin_fmaf((float)(acc[2][i] * 256 + acc[1][i]), 256.0f, (float)acc[0][i]);
        }
    }

    // The running maximum and sum over the 16 scores x of this lane, four of
    // each tile t, and their probabilities in fp16: 8 h .. 8 h + 7 in ph[h] (and
    // pl[h]).  f[t], vs[t]: factors of tile t's scores and values; keep(i): score
    // i counts (asked only when not `full`).
    template <typename Keep>
    __device__ __forceinline__ void softmax(float* x, const float* f, const float* vs, float vmax, bool full, Keep keep,
                                            v8h* ph, v8h* pl) {
        if (!full) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = keep(i) ? x[i] : kNegInf;
        }
        // (factors are never negative: a tile's largest score is that of its
        // largest x; no token gives -inf, or NaN at a factor of 0, which the
        // maximum leaves out)
        float mx = kNegInf;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            mx = fmaxf(mx, fmaxf(fmaxf(x[4 * t], x[4 * t + 1]), fmaxf(x[4 * t + 2], x[4 * t + 3])) * f[t]);
        }
        mx = column_max(mx);
        if (__any(mx > m + kSlack || vmax > ref)) {
            // the values' scales count relative to the largest so far, as a power of two
            const float ref_new = vmax > ref ? __uint_as_float(((__float_as_uint(vmax) >> 23) + 1) << 23) : ref;
            const float m_new = fmaxf(m, mx);
            base = m_new == kNegInf ? 0.0f : m_new;
            const float al = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - base);
            l *= al;
            const float ao = al * (ref / ref_new);
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= ao;
            m = m_new;
            ref = ref_new;
            unit = kPeak / ref;
        }
        // (fused: a score keeps the bits that the product would round off)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_fmaf(x[i], f[i >> 2], -base);
        if (__any(fabsf(base) >= kHuge)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fminf(x[i], kSlack);
        }
        uint32_t hi[8], lo[8];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float pf = vs[i >> 1] * unit;
            float p0 = __builtin_amdgcn_exp2f(x[2 * i]), p1 = __builtin_amdgcn_exp2f(x[2 * i + 1]);
            if (!full) {
                p0 = keep(2 * i) ? p0 : 0.0f;
                p1 = keep(2 * i + 1) ? p1 : 0.0f;
            }
            sum += p0 + p1;
            const float w0 = p0 * pf, w1 = p1 * pf;
            hi[i] = __builtin_bit_cast(uint32_t, v2h{(_Float16)w0, (_Float16)w1});
            if (PL == 2) {
                // the remainder is taken from the packed bits themselves: the
                // compiler may otherwise round the product to fp16 a second
                // time, fused, and the two disagree at ties
                asm("" : "+v"(hi[i]));
                const v2h h = __builtin_bit_cast(v2h, hi[i]);
                const v2h r = {(_Float16)__builtin_fmaf((float)h[0], -1.0f, w0), (_Float16)__builtin_fmaf((float)h[1], -1.0f, w1)};
                lo[i] = __builtin_bit_cast(uint32_t, r);
            }
        }
        l += sum;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            ph[h] = __builtin_bit_cast(v8h, v4i{(int)hi[4 * h], (int)hi[4 * h + 1], (int)hi[4 * h + 2], (int)hi[4 * h + 3]});
            if (PL == 2)
                pl[h] = __builtin_bit_cast(v8h, v4i{(int)lo[4 * h], (int)lo[4 * h + 1], (int)lo[4 * h + 2], (int)lo[4 * h + 3]});
        }
    }

    // O^T += V^T P^T of one 16-dimension tile and half of the step's tokens
    __device__ __forceinline__ void value(int d, v8h v, v8h ph, v8h pl) {
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[d], 0, 0, 0);
        if (PL == 2) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[d], 0, 0, 0);
    }
};

// Four codes as fp16: code + 128 as the low bits of 1024, less 1152.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t* out) {
    const v2h bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    const uint32_t u = w ^ 0x80808080u;
    out[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    out[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
}

__device__ __forceinline__ v4i ldg(const int8_t* p) { return *(const v4i*)p; }

// Page number of the 16 tokens at tok as the table has it (of the last page
// where tok is past it), and whether it is one.  Apart, and always a load: a
// branch around it would make a loop wait for every load it has under way.
__device__ __forceinline__ int page_of(const AttnParams& a, const int32_t* tab, int tok, int npages) {
    return tab[min((unsigned)tok >> a.shift, (unsigned)npages - 1)];
}

__device__ __forceinline__ bool has_page(const AttnParams& a, int id, int tok, int npages) {
    return (((unsigned)tok >> a.shift) < (unsigned)npages) & ((unsigned)id < (unsigned)a.pages);
}

// A page to read in any case: without a page the first one, and what is read
// is masked.
__device__ __forceinline__ int safe_page(const AttnParams& a, int id) { return (unsigned)id < (unsigned)a.pages ? id : 0; }

// Offset of a block of 16 tokens.
__device__ __forceinline__ long block_of(const AttnParams& a, int id, int tok, int kvh, int hd) {
    const long blocks = ((long)safe_page(a, id) * a.kv_heads + kvh) << (a.shift - 4);
    return (blocks + ((tok & ((1 << a.shift) - 1)) >> 4)) * (16 * hd);
}

// A row's columns and how the context of a tile of them is cut.
struct Cut {
    int steps, active, per;
};

__device__ __forceinline__ Cut cut_context(const AttnParams& a, int most) {
    Cut c;
    c.steps = (most + kStep - 1) / kStep;
    c.active = (c.steps + a.min_steps - 1) / a.min_steps;
    c.active = c.active < 1 ? 1 : (c.active > a.splits ? a.splits : c.active);
    c.per = (c.steps + c.active - 1) / c.active;
    if (c.per > 0) c.active = (c.steps + c.per - 1) / c.per;
    return c;
}

// This lane's column of a tile at column `col` of a request.
struct Column {
    bool valid;
    int row, head, limit;  // limit: tokens that it attends to

    __device__ __forceinline__ Column(const AttnParams& a, long col, long cols, int start, int kvh) {
        valid = col < cols;
        row = start + (valid ? (int)(col / a.group) : 0);
        head = kvh * a.group + (valid ? (int)(col % a.group) : 0);
        limit = 0;
        if (valid) {
            limit = a.positions[row] + 1;
            limit = limit < 0 ? 0 : (limit > a.max_context ? a.max_context : limit);
        }
    }
};

// out = o / l, zeros for a row that attends to nothing
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// Few columns (decode rows): the workgroup's four waves share 16 columns and
// take every fourth step of the part blockIdx.z of the context.  Bound by the
// cache's bytes: codes go straight to registers, each read once, the next
// step's under way while this one's are used.  (Row r of the key operand of
// tile t is token 16 (r >> 2) + 4 t + (r & 3): a lane's 16 scores are those of
// the 16 tokens whose values it holds, in one page.)  Seven contexts of 65536
// tokens, 5 heads of 128: 113 us, 5.2 TB/s; 64 rows of up to 4096 tokens 40 us,
// 4.7 TB/s.
template <int HD, int PL>
__global__ __launch_bounds__(256) void paged_attn_rows_kernel(AttnParams a) {
    using W = Wave<HD, PL>;
    constexpr int NS = W::NS, ND = W::ND;
    constexpr int LDO = HD + 4;
    __shared__ __align__(16) float o_s[4 * 16 * LDO];
    __shared__ float ml_s[4 * 16 * 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.y, part = blockIdx.z;
    // beside the chunk kernel a request has one tile here or none: no search
    int first_tile = blockIdx.x;
    const int r = a.hi_cols == 16 ? blockIdx.x : find_request(a, 16, blockIdx.x, lane, &first_tile);
    if (r < 0) return;
    int start = a.row_start[r], end = a.row_start[r + 1];
    start = start < 0 ? 0 : start;
    end = end > a.rows ? a.rows : end;
    const long cols = (long)(end - start) * a.group;
    const long c0 = (long)(blockIdx.x - first_tile) * 16;
    if (c0 >= cols || cols > a.hi_cols) return;
    const Column me(a, c0 + n, cols, start, kvh);
    int most = me.limit;
    int least = me.valid ? me.limit : 0x7fffffff;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) {
        most = max(most, __shfl_xor(most, d, 64));
        least = min(least, __shfl_xor(least, d, 64));
    }
    const Cut cut = cut_context(a, most);
    if (part >= cut.active) return;

    W w;
    w.clear();
    const int s1 = min((part + 1) * cut.per, cut.steps);
    const int first = part * cut.per + wave;
    if (first < s1) {
        const int32_t* tab = a.table + (long)r * a.max_pages;
        const int npages = (most + (1 << a.shift) - 1) >> a.shift;
        v4i k[4][NS], v[ND];
        float ks, vs;
        int pk, pv;  // pages of this lane's key row and of its 16 tokens
        auto pages = [&](int tok0) {
            pk = page_of(a, tab, tok0 + 16 * (n >> 2), npages);
            pv = page_of(a, tab, tok0 + 16 * g, npages);
        };
        auto keys = [&](int page, int tok0) {
            const int8_t* p = a.k + block_of(a, page, tok0 + 16 * (n >> 2), kvh, HD) + 256 * g + 16 * (n & 3);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    if (HD >= 64 || 16 * g < HD) k[t][s] = ldg(p + 64 * t + 1024 * s);
                    else k[t][s] = v4i{0, 0, 0, 0};
                }
            }
        };
        auto scales = [&](int page) {
            const long at = (long)safe_page(a, page) * a.kv_heads + kvh;
            ks = a.ks[at];
            vs = a.vs[at];
        };
        auto values = [&](int page, int tok0) {
            const int8_t* p = a.v + block_of(a, page, tok0 + 16 * g, kvh, HD) + 16 * n;
#pragma unroll
            for (int d = 0; d < ND; ++d) v[d] = ldg(p + 256 * d);
        };
        v8h ph[2], pl[2];
        auto finish = [&](float* x, float ks_, float vs_, bool ok, int tok0) {
            const float f = w.qf * ks_, fs[4] = {f, f, f, f};
            const float vo = ok ? vs_ : 0.0f, vv[4] = {vo, vo, vo, vo};
            const int left = ok ? me.limit - (tok0 + 16 * g) : 0;
            w.softmax(x, fs, vv, column_max(vo), tok0 + kStep <= least && __all(ok), [&](int i) { return i < left; }, ph, pl);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                uint32_t c[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) codes_f16((uint32_t)v[d][j], c + 2 * j);
                w.value(d, __builtin_bit_cast(v8h, v4i{(int)c[0], (int)c[1], (int)c[2], (int)c[3]}), ph[0], pl[0]);
                w.value(d, __builtin_bit_cast(v8h, v4i{(int)c[4], (int)c[5], (int)c[6], (int)c[7]}), ph[1], pl[1]);
            }
        };
        pages(first * kStep);
        keys(pk, first * kStep);
        scales(pv);
        values(pv, first * kStep);
        int pk1 = pk, pv1 = pv;
        pages((first + 4) * kStep);
        w.load_q(a, (long)me.row * a.q_stride + (long)me.head * HD, me.valid, g);
        // the next step's keys are on their way from the end of this step's
        // scores on, its values from the end of this step's product, its page
        // numbers a step earlier
        int s = first;
        float x[16];
        for (; s + 4 < s1; s += 4) {
#pragma unroll
            for (int t = 0; t < 4; ++t) w.tile(k[t], x + 4 * t);
            const float ks0 = ks, vs0 = vs;
            const bool ok = has_page(a, pv1, s * kStep + 16 * g, npages);
            pk1 = pk, pv1 = pv;
            keys(pk1, (s + 4) * kStep);
            scales(pv1);
            pages((s + 8) * kStep);
            finish(x, ks0, vs0, ok, s * kStep);
            values(pv1, (s + 4) * kStep);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) w.tile(k[t], x + 4 * t);
        finish(x, ks, vs, has_page(a, pv1, s * kStep + 16 * g, npages), s * kStep);
    }
    // join the four waves' parts
    const float l = column_sum(w.l), unit = w.ref / kPeak;
#pragma unroll
    for (int d = 0; d < ND; ++d) *(v4f*)&o_s[(wave * 16 + n) * LDO + 16 * d + 4 * g] = w.o[d] * unit;
    if (g == 0) {
        ml_s[(wave * 16 + n) * 2] = w.m;
        ml_s[(wave * 16 + n) * 2 + 1] = l;
    }
    __syncthreads();
    // thread t: column t / 16, dimensions 4 (t % 16) + 64 i
    const int cn = threadIdx.x >> 4, d0 = 4 * (threadIdx.x & 15);
    if (c0 + cn >= cols) return;
    float m = kNegInf;
    for (int i = 0; i < 4; ++i) m = fmaxf(m, ml_s[(i * 16 + cn) * 2]);
    float wt[4], sum = 0.0f;
    for (int i = 0; i < 4; ++i) {
        const float mi = ml_s[(i * 16 + cn) * 2];
        wt[i] = mi == m ? 1.0f : __builtin_amdgcn_exp2f(mi - m);
        sum += wt[i] * ml_s[(i * 16 + cn) * 2 + 1];
    }
    const int row = start + (int)((c0 + cn) / a.group), head = kvh * a.group + (int)((c0 + cn) % a.group);
    const long rh = (long)row * a.heads + head, all = (long)a.rows * a.heads;
    const float inv = cut.active == 1 ? inverse_sum(sum) : 1.0f;
    for (int d = d0; d < HD; d += 64) {
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < 4; ++i) {
            const v4f p = *(const v4f*)&o_s[(i * 16 + cn) * LDO + d];
            for (int j = 0; j < 4; ++j) y[j] += wt[i] * p[j];
        }
        for (int j = 0; j < 4; ++j) y[j] *= inv;
        if (cut.active == 1) store4(a.out, a.type, (long)row * a.out_stride + (long)head * HD + d, a.vec, y);
        else *(float4*)&a.part_o[(part * all + rh) * HD + d] = make_float4(y[0], y[1], y[2], y[3]);
    }
    if ((threadIdx.x & 15) == 0 && a.splits > 1) {
        if (cut.active > 1) {
            a.part_ml[(part * all + rh) * 2] = m;
            a.part_ml[(part * all + rh) * 2 + 1] = sum;
        }
        if (part == 0) a.active[rh] = cut.active;
    }
}

// Many columns of one request (chunks of prompts): four waves of 16 columns
// each go through the part's steps together.  Bound by vector instructions
// (about 15 for each score, exp2 among them), so what the waves can share is
// done once: a step's codes are staged in LDS, keys as stored, values as fp16,
// in the order of the operands (whole-line reads without bank conflicts), and
// few enough registers stay that three waves share a SIMD (head_dim up to 128;
// eight waves of 128 columns at four a SIMD spilled: 319 us).
// Row r of the key operand of tile t is token 16 t + r here: a lane's scores
// are tokens 16 t + 4 g + i, and the values' tokens are written in that order.
// Two buffers, one barrier a step.
constexpr int kChunkWaves = 4;
constexpr int kChunkCols = 16 * kChunkWaves;

// (Four prompts of 2048 tokens, 20 heads of 128, fp32: 255 us, 335 TFLOP/s; the
// same tiles with codes straight to registers 284.)
template <int HD, int PL>
__global__ __launch_bounds__(64 * kChunkWaves, HD <= 128 ? 3 : 1) void paged_attn_chunk_kernel(AttnParams a) {
    using W = Wave<HD, PL>;
    constexpr int NS = W::NS, ND = W::ND, THREADS = 64 * kChunkWaves;
    constexpr int KU = 4 * HD;                           // 16-byte units of a step's keys, and of its values
    constexpr int PER = (2 * KU + THREADS - 1) / THREADS;  // units of a thread
    struct Scales {
        float k[4], v[4];
        int ok;
        float vmax;
    };
    __shared__ v4i k_s[2][KU];
    __shared__ v4i v_s[2][2 * KU];
    __shared__ Scales sc_s[2];
    __shared__ int most_s[kChunkWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.y, part = blockIdx.z;
    int first_tile;
    // the last tiles of a chunk attend to the most: they start first
    const int x0 = gridDim.x - 1 - blockIdx.x;
    const int r = find_request(a, kChunkCols, x0, lane, &first_tile);
    if (r < 0) return;
    int start = a.row_start[r], end = a.row_start[r + 1];
    start = start < 0 ? 0 : start;
    end = end > a.rows ? a.rows : end;
    const long cols = (long)(end - start) * a.group;
    const long c0 = (long)(x0 - first_tile) * kChunkCols;
    if (c0 >= cols || cols <= a.hi_cols) return;
    const Column me(a, c0 + 16 * wave + n, cols, start, kvh);
    int mine = me.limit;
    int least = me.valid ? me.limit : 0x7fffffff;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) {
        mine = max(mine, __shfl_xor(mine, d, 64));
        least = min(least, __shfl_xor(least, d, 64));
    }
    if (lane == 0) most_s[wave] = mine;
    __syncthreads();
    int most = 0;
#pragma unroll
    for (int i = 0; i < kChunkWaves; ++i) most = max(most, most_s[i]);
    const Cut cut = cut_context(a, most);
    if (part >= cut.active) return;

    W w;
    w.clear();
    const int s0 = part * cut.per, s1 = min(s0 + cut.per, cut.steps);
    if (s0 < s1) {
        const int32_t* tab = a.table + (long)r * a.max_pages;
        const int npages = (most + (1 << a.shift) - 1) >> a.shift;
        // unit u of a step: keys (u < KU) or values, block (u % KU) / HD, 16 bytes
        // u % HD of it
        int page[PER], page_sc;
        v4i code[PER];
        float sk, sv;
        auto pages = [&](int tok0) {
#pragma unroll
            for (int i = 0; i < PER; ++i) page[i] = page_of(a, tab, tok0 + 16 * (((threadIdx.x + THREADS * i) % KU) / HD), npages);
            page_sc = page_of(a, tab, tok0 + 16 * (lane & 3), npages);
        };
        auto fetch = [&](int tok0) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int u = threadIdx.x + THREADS * i;
                if (2 * KU % THREADS == 0 || u < 2 * KU) {
                    const long at = block_of(a, page[i], tok0 + 16 * ((u % KU) / HD), kvh, HD) + 16 * (u % HD);
                    code[i] = ldg((u < KU ? a.k : a.v) + at);
                }
            }
            const long at = (long)safe_page(a, page_sc) * a.kv_heads + kvh;
            sk = a.ks[at];
            sv = a.vs[at];
        };
        auto stage = [&](int b, int sc_page, int tok0) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int u = threadIdx.x + THREADS * i;
                if (u < KU) {
                    k_s[b][u] = code[i];
                } else if (2 * KU % THREADS == 0 || u < 2 * KU) {
                    // dimension d of block t: its tokens 4 g .. are lane (d % 16, g)'s
                    const int t = (u - KU) / HD, d = (u - KU) % HD;
                    uint2* to = (uint2*)&v_s[b][((t >> 1) * ND + (d >> 4)) * 64 + (d & 15)] + (t & 1);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t c[2];
                        codes_f16((uint32_t)code[i][j], c);
                        to[j * 32] = make_uint2(c[0], c[1]);
                    }
                }
            }
            if (wave == kChunkWaves - 1) {
                const bool ok = has_page(a, sc_page, tok0 + 16 * (lane & 3), npages);
                const float v = ok ? sv : 0.0f;
                float vm = fmaxf(v, __shfl_xor(v, 1, 64));
                vm = fmaxf(vm, __shfl_xor(vm, 2, 64));
                const unsigned long long all = __ballot(ok);
                if (lane < 4) {
                    sc_s[b].k[lane] = sk;
                    sc_s[b].v[lane] = v;
                }
                if (lane == 0) {
                    sc_s[b].ok = (int)(all & 15);
                    sc_s[b].vmax = vm;
                }
            }
        };
        pages(s0 * kStep);
        fetch(s0 * kStep);
        int sc_page = page_sc;
        pages((s0 + 1) * kStep);
        w.load_q(a, (long)me.row * a.q_stride + (long)me.head * HD, me.valid, g);
        stage(0, sc_page, s0 * kStep);
        __syncthreads();
        const int my_steps = (mine + kStep - 1) / kStep;
        for (int s = s0; s < s1; ++s) {
            const int b = (s - s0) & 1;
            const bool more = s + 1 < s1;
            if (more) {
                fetch((s + 1) * kStep);
                sc_page = page_sc;
                pages((s + 2) * kStep);
            }
            if (s < my_steps) {
                float x[16];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    v4i k[NS];
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        if (HD >= 64 || 16 * g < HD) k[i] = k_s[b][t * HD + (g + 4 * i) * 16 + n];
                        else k[i] = v4i{0, 0, 0, 0};
                    }
                    w.tile(k, x + 4 * t);
                }
                const Scales& sc = sc_s[b];
                const int ok = sc.ok;
                const float f[4] = {w.qf * sc.k[0], w.qf * sc.k[1], w.qf * sc.k[2], w.qf * sc.k[3]};
                const float vs[4] = {sc.v[0], sc.v[1], sc.v[2], sc.v[3]};
                const int left = me.limit - (s * kStep + 4 * g);
                v8h ph[2], pl[2];
                w.softmax(x, f, vs, sc.vmax, s * kStep + kStep <= least && ok == 15,
                          [&](int i) { return 16 * (i >> 2) + (i & 3) < left && (ok >> (i >> 2) & 1); }, ph, pl);
                // operand reads kAhead ahead of the products that take them (left
                // alone, the compiler waits for each)
                constexpr int kAhead = 4;
                v4i vb[kAhead];
                auto operand = [&](int i) { return v_s[b][((i & 1) * ND + (i >> 1)) * 64 + lane]; };
#pragma unroll
                for (int i = 0; i < kAhead; ++i) vb[i] = operand(i);
#pragma unroll
                for (int i = 0; i < 2 * ND; ++i) {
                    const v4i v = vb[i % kAhead];
                    __builtin_amdgcn_sched_barrier(0);
                    w.value(i >> 1, __builtin_bit_cast(v8h, v), ph[i & 1], pl[i & 1]);
                    if (i + kAhead < 2 * ND) vb[i % kAhead] = operand(i + kAhead);
                }
            }
            if (more) stage(b ^ 1, sc_page, (s + 1) * kStep);
            __syncthreads();
        }
    }
    const float l = column_sum(w.l), unit = w.ref / kPeak;
    if (!me.valid) return;
    const long rh = (long)me.row * a.heads + me.head;
    if (cut.active == 1) {
        const float inv = inverse_sum(l) * unit;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            float y[4];
            for (int j = 0; j < 4; ++j) y[j] = w.o[d][j] * inv;
            store4(a.out, a.type, (long)me.row * a.out_stride + (long)me.head * HD + 16 * d + 4 * g, a.vec, y);
        }
    } else {
        const long at = (long)part * a.rows * a.heads + rh;
#pragma unroll
        for (int d = 0; d < ND; ++d) *(v4f*)&a.part_o[at * HD + 16 * d + 4 * g] = w.o[d] * unit;
        if (g == 0) {
            a.part_ml[at * 2] = w.m;
            a.part_ml[at * 2 + 1] = l;
        }
    }
    if (a.splits > 1 && part == 0 && g == 0) a.active[rh] = cut.active;
}

// Joins the parts of rows whose context was cut: one wave per (row, head).
template <int HD>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnParams a) {
    const int lane = threadIdx.x & 63;
    const long rh = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long all = (long)a.rows * a.heads;
    if (rh >= all) return;
    const int row = (int)(rh / a.heads), head = (int)(rh % a.heads);
    if (row >= a.row_start[a.requests] || row < a.row_start[0]) return;  // rows of no request: left as they are
    const int active = a.active[rh];
    if (active <= 1 || active > a.splits) return;
    float m = kNegInf, l = 0.0f;
    if (lane < active) {
        m = a.part_ml[(lane * all + rh) * 2];
        l = a.part_ml[(lane * all + rh) * 2 + 1];
    }
    float top = m;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, shfl_xor_f(top, d));
    const float wt = lane < active ? (m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top)) : 0.0f;
    float sum = wt * l;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += shfl_xor_f(sum, d);
    const float inv = inverse_sum(sum);
    constexpr int LW = HD / 4 < 64 ? HD / 4 : 64;  // lanes of one part's row
    constexpr int PAR = 64 / LW;                   // parts read at a time
    const int d = 4 * (lane % LW);
    v4f y = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < active; i += PAR) {
        const int p = i + lane / LW;
        const float wp = __shfl(wt, p < 64 ? p : 63, 64);
        if (p < active) y += wp * *(const v4f*)&a.part_o[(p * all + rh) * HD + d];
    }
#pragma unroll
    for (int s = 32; s >= LW; s >>= 1) {
        for (int j = 0; j < 4; ++j) y[j] += shfl_xor_f(y[j], s);
    }
    if (lane < LW) {
        float z[4];
        for (int j = 0; j < 4; ++j) z[j] = y[j] * inv;
        store4(a.out, a.type, (long)row * a.out_stride + (long)head * HD + d, a.vec, z);
    }
}

// Parts of a context: enough workgroups to fill the chip (two of four waves a
// CU) and even out ragged lengths; 512 and 1024 were a few per cent slower on
// decode rows, 2048 14 % (each part has its own start and join).
constexpr int kWantGroups = 768;
constexpr int kMinSteps = 4;  // 256 tokens: a step for each wave of a decode workgroup

static int splits_for(int rows, int heads, int kv_heads, int requests, int max_context) {
    const long tiles = ceil_div(rows * (heads / kv_heads), 64);
    const long groups = (tiles > requests ? tiles : (requests < rows ? requests : rows)) * kv_heads;
    long s = (kWantGroups + groups - 1) / groups;
    const long most = ceil_div(max_context, kMinSteps * kStep);
    s = s > most ? most : s;
    return (int)(s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : s));
}

struct PartLayout {
    size_t o, ml, active, bytes;
};

static PartLayout part_layout(int rows, int heads, int hd, int splits) {
    PartLayout p{0, 0, 0, 0};
    if (splits <= 1) return p;
    const size_t rh = (size_t)rows * heads;
    auto pad = [](size_t b) { return (b + 255) & ~(size_t)255; };
    p.ml = pad(rh * splits * hd * 4);
    p.active = p.ml + pad(rh * splits * 8);
    p.bytes = p.active + pad(rh * 4);
    return p;
}

size_t paged_attn_workspace(int rows, int heads, int kv_heads, int hd, int requests, int max_context) {
    return part_layout(rows, heads, hd, splits_for(rows, heads, kv_heads, requests, max_context)).bytes;
}

template <int HD, int PL>
static hipError_t launch_typed(AttnParams& a, hipStream_t s) {
    const long cols = (long)a.rows * a.group;
    // requests of at most 16 columns (decode rows) take the rows kernel; where
    // every request may be one, it takes all of them
    const bool few = cols <= 16l * a.requests;
    a.hi_cols = few ? 0x7fffffff : 16;
    hipLaunchKernelGGL((paged_attn_rows_kernel<HD, PL>),
                       dim3((unsigned)(few ? cols / 16 + a.requests : a.requests), (unsigned)a.kv_heads, (unsigned)a.splits),
                       dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!few) {
        hipLaunchKernelGGL((paged_attn_chunk_kernel<HD, PL>),
                           dim3((unsigned)(cols / kChunkCols + a.requests), (unsigned)a.kv_heads, (unsigned)a.splits),
                           dim3(64 * kChunkWaves), 0, s, a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (a.splits > 1) {
        hipLaunchKernelGGL(paged_attn_join_kernel<HD>, dim3((unsigned)(((long)a.rows * a.heads + 3) / 4)), dim3(256), 0, s, a);
        e = hipGetLastError();
    }
    return e;
}

hipError_t launch_paged_attn(const PagedAttn& p, hipStream_t s) {
    AttnParams a{};
    a.k = p.c.k;
    a.v = p.c.v;
    a.ks = p.c.k_scale;
    a.vs = p.c.v_scale;
    a.table = p.table;
    a.row_start = p.row_start;
    a.positions = p.positions;
    a.q = p.q;
    a.out = p.out;
    a.pages = p.c.pages;
    a.shift = __builtin_ctz((unsigned)p.c.page);
    a.kv_heads = p.c.kv_heads;
    a.max_pages = p.max_pages;
    a.requests = p.requests;
    a.rows = p.rows;
    a.heads = p.heads;
    a.group = p.heads / p.c.kv_heads;
    a.type = p.type;
    a.max_context = p.max_context;
    a.min_steps = kMinSteps;
    a.q_stride = p.q_stride;
    a.out_stride = p.out_stride;
    a.scale2 = p.scale * 1.44269504088896340736f;
    const int size = p.type == ROW_BF16 ? 2 : (p.type == ROW_F32 ? 4 : 8);
    a.vec = p.type != ROW_F64 && ((uintptr_t)p.q & 15) == 0 && ((uintptr_t)p.out & 15) == 0 &&
            (p.q_stride * size) % 16 == 0 && (p.out_stride * size) % 16 == 0;
    a.splits = splits_for(p.rows, p.heads, p.c.kv_heads, p.requests, p.max_context);
    const PartLayout l = part_layout(p.rows, p.heads, p.c.hd, a.splits);
    a.part_o = (float*)((char*)p.workspace + l.o);
    a.part_ml = (float*)((char*)p.workspace + l.ml);
    a.active = (int32_t*)((char*)p.workspace + l.active);
#define ATTN(HD) \
    case HD: return p.type == ROW_BF16 ? launch_typed<HD, 1>(a, s) : launch_typed<HD, 2>(a, s);
    switch (p.c.hd) {
        ATTN(32)
        ATTN(64)
        ATTN(128)
        ATTN(256)
        default: return hipErrorInvalidValue;
    }
#undef ATTN
}

}  // namespace lamd
