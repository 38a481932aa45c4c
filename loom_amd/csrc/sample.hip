// sample.hip -- one token per row of logits from a given random number, with
// temperature, top-k, top-p and min-p.
//
// With w_i = exp((l_i - max) / T) and the tokens ranked by value (equal values
// by index), each filter keeps a first part of the ranking:
//   top-k  the first k
//   top-p  the shortest part of those whose mass reaches p of theirs
//   min-p  the tokens with w >= min_p
// and the token is the first in vocabulary order whose kept mass, summed from
// token 0, exceeds u times the whole.  No row is sorted: a histogram over
// w's logarithm gives the count and mass of every 1/32 of a nat, and a filter's
// end or the token itself is then looked for in one bucket.
//
// Masses are sums of integers (fixed point) or of fp64 values in a fixed
// order, so a row's token does not depend on the order of atomics.  A token
// more than 32 nats under the row's largest (w < 1.3e-14) has no mass.
#include "paged.hpp"

namespace lamd {

constexpr int kThreads = 1024;
constexpr int kSeg = 8192;       // tokens of a segment: eight per thread
constexpr int kBuckets = 1024;   // 32 nats
constexpr double kPerNat = 32.0;
constexpr int kList = 1024;      // a bucket of up to so many tokens is ranked directly
constexpr int kMaxSegs = 1024;
constexpr double kFar = 0x1p35;  // |32 max / T| from which neighbouring floats are over 32 nats apart
constexpr double kBig = 0x1p15;  // and from which the product's low part counts
// Masses of the histogram and of single tokens differ by under 2^-39 of the
// whole; where the definition compares equal sums (equal logits), they must
// compare equal: a sum within this part of the whole counts as equal.
constexpr double kSame = 0x1p-37;
constexpr double kDefUnit = 0x1p39;
constexpr double kMassUnit = 0x1p48;
constexpr unsigned long long kDefMask = (1ull << 48) - 1;

struct SegMax {
    float value;  // -inf: no token of the segment can be drawn
    int index;
    int listed;   // tokens of its list
};

__device__ __forceinline__ float usable(float x) {  // NaN: never drawn; +inf: the largest finite value
    return fminf(fmaxf(x, -__builtin_inff()), 3.402823466e38f);
}

// Order of values as unsigned integers.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 counts as +0)
    return (u >> 31) ? ~u : u | 0x80000000u;
}

struct Better {
    __device__ __forceinline__ static bool before(float a, int ia, float b, int ib) {
        return a > b || (a == b && ia < ib);
    }
};

// Largest over the wave, in every lane: rotations within rows of 16, then the
// exchanges of rows and halves.
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = dpp_max<0x128>(v);
    v = dpp_max<0x124>(v);
    v = dpp_max<0x122>(v);
    v = dpp_max<0x121>(v);
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Largest value (lowest index of equal ones) over the workgroup.
__device__ __forceinline__ void block_best(float& v, int& i, float* sv, int* si) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const float ov = __shfl_xor(v, d, 64);
        const int oi = __shfl_xor(i, d, 64);
        if (Better::before(ov, oi, v, i)) v = ov, i = oi;
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) sv[wave] = v, si[wave] = i;
    __syncthreads();
    v = sv[0], i = si[0];
    for (int w = 1; w < kThreads / 64; ++w) {
        if (Better::before(sv[w], si[w], v, i)) v = sv[w], i = si[w];
    }
    __syncthreads();
}

// z = l / T on the absolute grid of 1/32 nats: t = 32 z, its bucket b.
struct Place {
    double t, b;
};

__device__ __forceinline__ Place place(float l, double per_t) {  // per_t = 32 / T
    Place p;
    p.t = (double)l * per_t;
    p.b = floor(p.t);
    return p;
}

// Bucket of l under a largest value's (at distance d from it, or kBuckets when
// it is too far to have a mass).
__device__ __forceinline__ int bucket_of(const Place& p, const Place& top) {
    const double d = top.b - p.b;
    if (fabs(top.t) >= kFar) return p.t == top.t ? 0 : kBuckets;
    return d < (double)kBuckets ? (int)d : kBuckets;
}

// What the rounded product t leaves off (counts from |t| = kBig on).
__device__ __forceinline__ double low_part(float l, double per_t, double t) { return __builtin_fma((double)l, per_t, -t); }

// (1 - exp(r / 32)) * 2^39 as an integer, for r in [-1, 0]: Taylor, the first
// term left out is under 1.3e-12; the sum with 2^52 leaves the integer in the
// low bits.
__device__ __forceinline__ unsigned long long deficit(double r) {
    constexpr double h = 1.0 / 32.0, u = 0x1p39;
    double y = -u * h * h * h * h * h / 120.0;
    y = __builtin_fma(y, r, -u * h * h * h * h / 24.0);
    y = __builtin_fma(y, r, -u * h * h * h / 6.0);
    y = __builtin_fma(y, r, -u * h * h / 2.0);
    y = __builtin_fma(y, r, -u * h);
    y = __builtin_fma(y, r, 0x1p52);
    return (unsigned long long)__double_as_longlong(y) & ((1ull << 52) - 1);
}

// Four consecutive logits of a row at i (i % 4 == 0), -inf past the end.
__device__ __forceinline__ float4 load4(const float* row, int vocab, int i, bool vec) {
    if (vec && i + 4 <= vocab) return *(const float4*)(row + i);
    float4 f;
    f.x = i < vocab ? row[i] : -__builtin_inff();
    f.y = i + 1 < vocab ? row[i + 1] : -__builtin_inff();
    f.z = i + 2 < vocab ? row[i + 2] : -__builtin_inff();
    f.w = i + 3 < vocab ? row[i + 3] : -__builtin_inff();
    return f;
}

struct SampleParams {
    const float* logits;
    long stride;
    int vocab, segs;
    bool vec;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int32_t* ids;
    SegMax* seg_max;            // [row][seg]
    unsigned long long* hist;   // [row][seg][kBuckets]: count << 48 | deficits
    uint16_t* first;            // [row][seg][kBuckets]: where a bucket's tokens start in the list
    uint16_t* list;             // [row][seg][kSeg]: tokens (within the segment) by bucket
};

struct Filters {
    float temperature, top_p, min_p;
    int top_k;

    __device__ __forceinline__ Filters(const SampleParams& a, long row) {
        temperature = a.temperature ? a.temperature[row] : 1.0f;
        top_k = a.top_k ? a.top_k[row] : 0;
        top_p = a.top_p ? a.top_p[row] : 1.0f;
        min_p = a.min_p ? a.min_p[row] : 0.0f;
    }
    __device__ __forceinline__ bool any(int vocab) const {
        return (top_k > 0 && top_k < vocab) || top_p < 1.0f || min_p > 0.0f;
    }
};

// v of another lane of the wave (CTRL), 0 where there is none or the row is not
// in ROWS.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_of(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    } else {
        const long long b = __builtin_bit_cast(long long, v);
        const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xf, false);
        const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (long long)(((unsigned long long)(uint32_t)hi << 32) | (uint32_t)lo));
    }
}

// Inclusive sums in lane order (row_shr 1, 2, 4, 8, then the rows' last lanes).
template <typename T>
__device__ __forceinline__ T row_scan(T v) {
    v += dpp_of<0x111, 0xf>(v);
    v += dpp_of<0x112, 0xf>(v);
    v += dpp_of<0x114, 0xf>(v);
    v += dpp_of<0x118, 0xf>(v);
    return v;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v = row_scan(v);
    v += dpp_of<0x142, 0xa>(v);
    v += dpp_of<0x143, 0xc>(v);
    return v;
}

// Inclusive sums over the workgroup in thread order, and their total.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* wave_sum, T* total) {
    static_assert(kThreads == 1024, "one row of lanes scans the waves' sums");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) wave_sum[wave] = v;
    __syncthreads();
    const T all = row_scan(wave_sum[lane & 15]);
    *total = __shfl(all, 15, 64);
    const T before = __shfl(all, wave > 0 ? wave - 1 : 0, 64);
    return wave > 0 ? v + before : v;
}

// One workgroup per (segment, row): its largest value, its histogram relative
// to it, and (where a filter may ask) its tokens listed by bucket.  A bucket's
// mass is kept as count and sum of 1 - exp(distance to the bucket's upper
// edge), one 64-bit LDS atomic a token, which is exact in any order and needs
// the row's maximum only when segments are joined; the atomic's old count is
// the token's place in its bucket's list.  Bound by vector instructions (about
// 25 a token, most fp64) and the atomics: 256 rows of 128256 tokens 60 us, 2.2
// TB/s of logits.
__global__ __launch_bounds__(kThreads) void sample_segments_kernel(SampleParams a) {
    __shared__ unsigned long long hist[kBuckets];
    __shared__ uint16_t first[kBuckets];
    __shared__ __align__(16) uint16_t list[kSeg];
    __shared__ float sv[kThreads / 64];
    __shared__ int si[kThreads / 64], at_s;
    const int tid = threadIdx.x, seg = blockIdx.y;
    const long row = blockIdx.x;
    const float* x = a.logits + row * a.stride;
    float l[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float4 f = load4(x, a.vocab, seg * kSeg + 4 * tid + j * 4 * kThreads, a.vec);
        l[4 * j] = usable(f.x), l[4 * j + 1] = usable(f.y), l[4 * j + 2] = usable(f.z), l[4 * j + 3] = usable(f.w);
    }
    hist[tid] = 0;
    const Filters fl(a, row);
    float best = l[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) best = fmaxf(best, l[i]);
    best = wave_max(best);
    if ((tid & 63) == 0) sv[tid >> 6] = best;
    if (tid == 0) at_s = 0x7fffffff;
    __syncthreads();
    best = sv[tid & (kThreads / 64 - 1)];
    best = wave_max(best);
    const long slot = row * a.segs + seg;
    const bool draws = fl.temperature > 0.0f && best > -__builtin_inff();
    if (!draws) {  // greedy, or nothing to draw: the first of the largest is all
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            if (l[i] == best) atomicMin(&at_s, seg * kSeg + 4 * tid + (i >> 2) * 4 * kThreads + (i & 3));
        }
        __syncthreads();
        if (tid == 0) a.seg_max[slot] = SegMax{best, at_s, 0};
        return;
    }
    const double per_t = kPerNat / (double)fl.temperature;
    const Place top = place(best, per_t);
    const bool far = fabs(top.t) >= kFar, big = fabs(top.t) >= kBig;
    int place_of[8];  // bucket << 16 | place in it
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        place_of[i] = -1;
        if (l[i] == -__builtin_inff()) continue;
        const Place p = place(l[i], per_t);
        int d;
        double r = (p.t - p.b) - 1.0;
        if (big) {  // (uniform)
            d = bucket_of(p, top);
            r = far ? 0.0 : fmin(fmax(r + low_part(l[i], per_t, p.t), -1.0), 0.0);
        } else {
            d = (int)(top.b - p.b);
        }
        if (d >= kBuckets) continue;
        const unsigned long long old = atomicAdd(&hist[d], (1ull << 48) | deficit(r));
        place_of[i] = d << 16 | (int)(old >> 48);
    }
    __syncthreads();
    const unsigned long long h = hist[tid];
    a.hist[slot * kBuckets + tid] = h;
    int listed = 0;
    if (fl.any(a.vocab)) {
        const int n = (int)(h >> 48);
        const int end = block_scan(n, si, &listed);
        first[tid] = (uint16_t)(end - n);
        a.first[slot * kBuckets + tid] = (uint16_t)(end - n);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (place_of[i] >= 0) {
                list[first[place_of[i] >> 16] + (place_of[i] & 0xffff)] =
                    (uint16_t)(4 * tid + (i >> 2) * 4 * kThreads + (i & 3));
            }
        }
        __syncthreads();
        if (8 * tid < listed) ((uint4*)(a.list + slot * kSeg))[tid] = ((const uint4*)list)[tid];
    }
    if (tid == 0) a.seg_max[slot] = SegMax{best, seg * kSeg, listed};
}

// What a row keeps: buckets up to `bucket`, and of those the tokens ranked at
// or before (key, index).
struct Cut {
    int bucket;
    uint32_t key;
    int index;
};

struct PickShared {
    double factor[kBuckets];   // exp(upper edge of a bucket - max)
    double mass[kBuckets];     // mass of the buckets up to here
    int count[kBuckets];
    unsigned long long list_w[kList];
    uint32_t list_key[kList];
    int list_idx[kList];
    unsigned long long part[kMaxSegs];  // kept mass of the cut's bucket by segment
    double seg_mass[kMaxSegs];
    int shift[kMaxSegs];  // a segment's buckets start so many below the row's (kBuckets: none)
    double wave_d[kThreads / 64];
    long long wave_i[kThreads / 64];
    float sv[kThreads / 64];
    int si[kThreads / 64];
    int n, found_i, found_j;
    uint32_t found_key, lo_key, hi_key;
    unsigned long long lo_ord, hi_ord, list_ord[64];
    double found_mass;
};

struct Row {
    const float* x;
    int vocab, segs;
    bool vec;
    double inv_t, per_t;  // 1 / T, 32 / T
    float max;
    Place top;
    const SegMax* seg_max;
    const unsigned long long* hist;
    const uint16_t* first;
    const uint16_t* list;

    __device__ __forceinline__ double weight(float l) const {
        return exp(((double)l - (double)max) * inv_t);
    }
    __device__ __forceinline__ unsigned long long fixed(float l) const {
        return (unsigned long long)(weight(l) * kMassUnit + 0.5);
    }
    __device__ __forceinline__ int bucket(float l) const { return bucket_of(place(l, per_t), top); }

    // f(value, key, index) for the row's tokens in buckets b0..b1 that the cut
    // keeps, from the segments' lists: a wave a segment
    template <typename F>
    __device__ __forceinline__ void each(const PickShared& s, int b0, int b1, const Cut& cut, F f) const {
        for (int i = threadIdx.x >> 6; i < segs; i += kThreads / 64) {
            const int shift = s.shift[i];
            const int d0 = b0 > shift ? b0 - shift : 0, d1 = b1 - shift;
            if (d1 < 0 || shift >= kBuckets) continue;
            const int from = first[(long)i * kBuckets + d0];
            const int to = d1 + 1 < kBuckets ? first[(long)i * kBuckets + d1 + 1] : seg_max[i].listed;
            for (int j = from + (threadIdx.x & 63); j < to; j += 64) {
                const int idx = i * kSeg + list[(long)i * kSeg + j];
                const float l = usable(x[idx]);
                const uint32_t k = key_of(l);
                if (k > cut.key || (k == cut.key && idx <= cut.index)) f(l, k, idx);
            }
        }
    }
};

// Where in buckets b0..b1 (of n tokens by the histogram) the ranking reaches
// `count` tokens (count > 0) or, with count = 0, the mass `target`, `before`
// being the mass of the buckets above b0.  Narrows the cut to that token,
// leaves the kept tokens of these buckets in s.part by segment and returns the
// mass kept in all.
__device__ double resolve(const Row& row, PickShared& s, int b0, int b1, long long n, long long count, double target,
                          double before, Cut* cut) {
    const int tid = threadIdx.x;
    uint32_t k0 = 0, k1 = 0xffffffffu;  // keys still in question
    double above = before;              // mass of what ranks before them
    long long left = count;             // tokens still to take
    for (int i = tid; i < kMaxSegs; i += kThreads) s.part[i] = 0;
    bool narrowed = false;
    while (n > kList) {
        narrowed = true;
        // keys of the tokens in question
        if (tid == 0) s.lo_key = 0xffffffffu, s.hi_key = 0;
        s.list_w[tid] = 0;
        s.list_idx[tid] = 0;
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        row.each(s, b0, b1, *cut, [&](float, uint32_t k, int) {
            if (k >= k0 && k <= k1) lo = min(lo, k), hi = max(hi, k);
        });
        if (lo <= hi) atomicMin(&s.lo_key, lo), atomicMax(&s.hi_key, hi);
        __syncthreads();
        lo = s.lo_key, hi = s.hi_key;
        if (lo >= hi) {
            k0 = lo, k1 = hi;
            break;
        }
        const int bits = 32 - __builtin_clz(hi - lo);
        const int shift = bits > 10 ? bits - 10 : 0;
        row.each(s, b0, b1, *cut, [&](float l, uint32_t k, int) {
            if (k < k0 || k > k1) return;
            const int at = (int)((hi - k) >> shift);
            atomicAdd(&s.list_idx[at], 1);
            atomicAdd(&s.list_w[at], (unsigned long long)(row.weight(l) * 0x1p40 + 0.5));
        });
        __syncthreads();
        const int c = s.list_idx[tid];
        const double w = (double)s.list_w[tid] * 0x1p-40;
        long long tc;
        double tw;
        const long long ci = block_scan<long long>(c, s.wave_i, &tc);
        const double wi = block_scan<double>(w, s.wave_d, &tw) + above;
        if (tid == 0) s.found_j = kThreads;
        __syncthreads();
        const bool crossed = c > 0 && (count ? ci >= left : wi >= target);
        if (crossed) atomicMin(&s.found_j, tid);
        __syncthreads();
        // (mass a rounding short of the target: the last of them)
        int at = s.found_j;
        if (at == kThreads) {
            __syncthreads();
            if (tid == 0) s.found_j = -1;
            __syncthreads();
            if (c > 0) atomicMax(&s.found_j, tid);
            __syncthreads();
            at = s.found_j;
        }
        if (tid == at) {
            s.found_mass = wi - w;
            s.found_i = c;
            s.wave_i[0] = ci - c;
        }
        __syncthreads();
        above = s.found_mass;
        n = s.found_i;
        left -= s.wave_i[0];
        __syncthreads();
        k1 = hi - ((uint32_t)at << shift);
        const uint32_t width = (1u << shift) - 1;
        k0 = k1 - width > k1 || k1 - width < lo ? lo : k1 - width;
    }
    if (n > kList) {
        // equal values: the token is the left-th of them by index
        const float l = __uint_as_float((k1 >> 31) ? (k1 & 0x7fffffffu) : ~k1);
        const double w = row.weight(l);
        if (!count) {
            const double want = ceil((target - above) / w);
            left = want < 1.0 ? 1 : (want > (double)n ? n : (long long)want);
        }
        const int last = k1 == cut->key ? cut->index : 0x7fffffff;
        long long seen = 0;
        if (tid == 0) s.found_i = last;
        __syncthreads();
        for (int base = 0; base < row.vocab && seen < left; base += 4 * kThreads) {
            const float4 v = load4(row.x, row.vocab, base + 4 * tid, row.vec);
            const float e[4] = {v.x, v.y, v.z, v.w};
            int c = 0;
            for (int i = 0; i < 4; ++i) c += usable(e[i]) == l && base + 4 * tid + i <= last;
            long long all;
            const long long upto = block_scan<long long>(c, s.wave_i, &all) + seen;
            if (upto >= left && upto - c < left) {
                long long have = upto - c;
                for (int i = 0; i < 4; ++i) {
                    if (usable(e[i]) == l && ++have == left) s.found_i = base + 4 * tid + i;
                }
            }
            seen += all;
        }
        __syncthreads();
        cut->key = k1;
        cut->index = s.found_i;
        above += (double)left * w;
    } else {
        if (tid == 0) s.n = 0;
        __syncthreads();
        row.each(s, b0, b1, *cut, [&](float l, uint32_t k, int idx) {
            if (k < k0 || k > k1) return;
            const int at = atomicAdd(&s.n, 1);
            if (at < kList) s.list_key[at] = k, s.list_idx[at] = idx, s.list_w[at] = row.fixed(l);
        });
        __syncthreads();
        const int m = s.n < kList ? s.n : kList;
        // a token a thread, its place in the ranking as one number (value, then
        // index); narrowed by histograms of 1024 parts until a wave's worth is
        // left to be ranked one against the other
        const uint32_t key = s.list_key[tid];
        const int idx = s.list_idx[tid];
        const unsigned long long w = s.list_w[tid];
        const unsigned long long ord = (unsigned long long)~key << 32 | (uint32_t)idx;
        bool open = tid < m;
        int now = m;
        unsigned long long done = 0;  // mass of tokens that rank before the open ones
        while (now > 64) {
            __syncthreads();
            if (tid == 0) s.lo_ord = ~0ull, s.hi_ord = 0;
            s.list_w[tid] = 0;
            s.list_idx[tid] = 0;
            __syncthreads();
            if (open) atomicMin(&s.lo_ord, ord), atomicMax(&s.hi_ord, ord);
            __syncthreads();
            const unsigned long long lo = s.lo_ord;
            const int bits = 64 - __builtin_clzll(s.hi_ord - lo);  // (over 64 tokens: never equal)
            const int shift = bits > 10 ? bits - 10 : 0;
            const int at = (int)((ord - lo) >> shift);
            if (open) {
                atomicAdd(&s.list_idx[at], 1);
                atomicAdd(&s.list_w[at], w);
            }
            __syncthreads();
            const int c = s.list_idx[tid];
            const unsigned long long cw = s.list_w[tid];
            long long tc, tw;
            const long long ci = block_scan<long long>(c, s.wave_i, &tc);
            const long long wi = block_scan<long long>((long long)cw, s.wave_i, &tw) + (long long)done;
            if (tid == 0) s.found_j = kThreads, s.found_i = 0;
            __syncthreads();
            if (c > 0) {
                if (count ? ci >= left : above + (double)wi * (1.0 / kMassUnit) >= target) atomicMin(&s.found_j, tid);
                atomicMax(&s.found_i, tid);  // (mass a rounding short of the target: the last)
            }
            __syncthreads();
            const int b = s.found_j < kThreads ? s.found_j : s.found_i;
            __syncthreads();
            if (tid == b) {
                s.n = c;
                s.lo_ord = (unsigned long long)(wi - (long long)cw);
                s.wave_i[0] = ci - c;
            }
            __syncthreads();
            now = s.n;
            done = s.lo_ord;
            left -= s.wave_i[0];
            open = open && at == b;
        }
        __syncthreads();
        if (tid == 0) s.n = 0, s.found_j = -1;
        __syncthreads();
        if (open) {
            const int at = atomicAdd(&s.n, 1);
            s.list_ord[at] = ord;
            s.list_w[at] = w;
        }
        __syncthreads();
        if (open) {
            int rank = 0;
            unsigned long long mass = done;
            for (int j = 0; j < now; ++j) {
                const bool b = s.list_ord[j] < ord;
                rank += b;
                mass += b ? s.list_w[j] : 0;
            }
            const double b = above + (double)mass * (1.0 / kMassUnit), e = above + (double)(mass + w) * (1.0 / kMassUnit);
            const bool here = count ? rank + 1 == left : (b < target || rank == 0) && (e >= target || rank + 1 == now);
            if (here) {
                s.found_key = key;
                s.found_i = idx;
                s.found_mass = e;
                s.found_j = 0;
            }
        }
        __syncthreads();
        if (s.found_j == 0) {
            cut->key = s.found_key;
            cut->index = s.found_i;
            above = s.found_mass;
        }
        __syncthreads();
        if (!narrowed && tid < m && (key > cut->key || (key == cut->key && idx <= cut->index))) {
            atomicAdd(&s.part[idx / kSeg], w);
        }
    }
    if (narrowed) {
        row.each(s, b0, b1, *cut, [&](float l, uint32_t, int idx) { atomicAdd(&s.part[idx / kSeg], row.fixed(l)); });
    }
    cut->bucket = b1;
    __syncthreads();
    return above;
}

// The whole of a row whose filters leave only tokens of buckets 0..b, n <=
// kFew of them: each ranked against the others, then summed by index.
// `whole` is the mass that top-p refers to where top-k is off.
constexpr int kFew = 256;

__device__ void pick_few(const Row& row, PickShared& s, int b, int n, const Filters& fl, bool kon, double whole,
                         float uniform, int* id) {
    const int tid = threadIdx.x;
    if (tid == 0) {
        s.n = 0;
        s.lo_ord = s.hi_ord = 0;  // masses of the first k, and of what is kept
        s.found_i = -1;
        s.found_j = 0x7fffffff;
    }
    __syncthreads();
    const Cut all{kBuckets - 1, 0u, 0x7fffffff};
    row.each(s, 0, b, all, [&](float l, uint32_t k, int idx) {
        const int at = atomicAdd(&s.n, 1);
        if (at < kFew) s.list_key[at] = k, s.list_idx[at] = idx, s.list_w[at] = row.fixed(l);
    });
    __syncthreads();
    n = s.n < kFew ? s.n : kFew;
    const bool mine = tid < n;
    uint32_t key = 0;
    int idx = 0, rank = 0;
    unsigned long long w = 0, before = 0;
    const int k = kon ? fl.top_k : 0x7fffffff;
    if (mine) {
        key = s.list_key[tid], idx = s.list_idx[tid], w = s.list_w[tid];
        for (int j = 0; j < n; ++j) {
            const uint32_t kj = s.list_key[j];
            const bool first = kj > key || (kj == key && s.list_idx[j] < idx);
            rank += first;
            before += first ? s.list_w[j] : 0;
        }
        if (rank < k) atomicAdd(&s.lo_ord, w);
    }
    __syncthreads();
    const double of = kon ? (double)s.lo_ord * (1.0 / kMassUnit) : whole;
    const double p = (double)fl.top_p, mp = fmin((double)fl.min_p, 1.0);
    bool keep = mine && rank < k;
    if (keep && rank > 0) {
        if (p < 1.0) keep = (double)before * (1.0 / kMassUnit) < p * of - kSame * of;
        if (mp > 0.0) {
            const uint32_t v = (key >> 31) ? (key & 0x7fffffffu) : ~key;
            keep = keep && row.weight(__uint_as_float(v)) >= mp;
        }
    }
    if (mine) s.list_w[tid] = keep ? w : 0;
    if (keep) {
        atomicAdd(&s.hi_ord, w);
        if (w > 0) atomicMax(&s.found_i, idx);
    }
    __syncthreads();
    const double kept = (double)s.hi_ord, u = (double)uniform;
    const double goal = u > 0.0 ? u * kept + kSame * kept : 0.0;
    if (keep && w > 0) {
        unsigned long long upto = 0;
        for (int j = 0; j < n; ++j) upto += s.list_idx[j] <= idx ? s.list_w[j] : 0;
        if ((double)upto > goal) atomicMin(&s.found_j, idx);
    }
    __syncthreads();
    if (tid == 0) *id = s.found_j != 0x7fffffff ? s.found_j : s.found_i;
}

// First bucket whose running count (mass) reaches the target.
template <typename F>
__device__ __forceinline__ int first_bucket(PickShared& s, F reached) {
    __syncthreads();
    if (threadIdx.x == 0) s.found_j = kBuckets - 1;
    __syncthreads();
    if (reached((int)threadIdx.x)) atomicMin(&s.found_j, (int)threadIdx.x);
    __syncthreads();
    const int b = s.found_j;
    __syncthreads();
    return b;
}

// One workgroup per row.  Bound by the latency of its steps, each a few loads
// from the lists or a scan, one after another: 27 us for a row whose filters
// leave few tokens, 43 us for 256 rows of a nucleus at once.
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleParams a) {
    __shared__ PickShared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long r = blockIdx.x;
    const SegMax* sm = a.seg_max + r * a.segs;
    const Filters fl(a, r);
    float best = -__builtin_inff();
    int at = 0x7fffffff;
    for (int i = tid; i < a.segs; i += kThreads) {
        const SegMax m = sm[i];
        if (Better::before(m.value, m.index, best, at)) best = m.value, at = m.index;
    }
    block_best(best, at, s.sv, s.si);
    Row row;
    row.x = a.logits + r * a.stride;
    row.vocab = a.vocab;
    row.segs = a.segs;
    row.vec = a.vec;
    if (!(fl.temperature > 0.0f) || best == -__builtin_inff()) {
        // greedy as loom_amd_greedy_sample: 0 when the first logit is NaN
        if (tid == 0) a.ids[r] = best == -__builtin_inff() || (!(fl.temperature > 0.0f) && row.x[0] != row.x[0]) ? 0 : at;
        return;
    }
    row.inv_t = 1.0 / (double)fl.temperature;
    row.max = best;
    row.per_t = kPerNat / (double)fl.temperature;
    row.top = place(best, row.per_t);
    row.seg_max = sm;
    row.hist = a.hist + r * a.segs * kBuckets;
    row.first = a.first + r * a.segs * kBuckets;
    row.list = a.list + r * a.segs * kSeg;
    const bool far = fabs(row.top.t) >= kFar;

    // the segments' histograms on the row's grid
    for (int i = tid; i < a.segs; i += kThreads) {
        const float v = sm[i].value;
        s.shift[i] = v == -__builtin_inff() ? kBuckets : bucket_of(place(v, row.per_t), row.top);
    }
    __syncthreads();
    unsigned long long def = 0;
    int cnt = 0;
#pragma unroll 8
    for (int i = 0; i < a.segs; ++i) {
        const int d = tid - s.shift[i];
        const unsigned long long h = d >= 0 ? row.hist[(long)i * kBuckets + d] : 0;
        cnt += (int)(h >> 48);
        def += h & kDefMask;
    }
    // a bucket's upper edge under the maximum, in 1/32 nats
    const double edge = far ? (tid == 0 ? 0.0 : -1e30)
                            : ((row.top.b - tid + 1.0) - row.top.t) - low_part(best, row.per_t, row.top.t);
    const double factor = exp(edge / kPerNat);
    s.factor[tid] = factor;
    long long tokens;
    double whole;
    const long long cum_n = block_scan<long long>(cnt, s.wave_i, &tokens);
    const double own = ((double)cnt - (double)def * (1.0 / kDefUnit)) * factor;
    const double cum_w = block_scan<double>(own, s.wave_d, &whole);
    s.count[tid] = (int)cum_n;
    s.mass[tid] = cum_w;
    __syncthreads();

    Cut cut{kBuckets - 1, 0u, 0x7fffffff};
    double kept = whole;
    int full = kBuckets;  // buckets below this one are kept whole; the rest of what is kept is in s.part
    auto count_before = [&](int b) { return b > 0 ? s.count[b - 1] : 0; };
    auto mass_before = [&](int b) { return b > 0 ? s.mass[b - 1] : 0.0; };

    const long long k = fl.top_k;
    if (fl.any(a.vocab)) {
        // the last bucket that any filter leaves tokens in (top-p of top-k needs
        // all of the first k)
        const bool kon = k > 0 && k < tokens;
        const double target = (double)fl.top_p * whole - kSame * whole, least = fmin((double)fl.min_p, 1.0) * (1.0 - 1e-9);
        const int b = first_bucket(s, [&](int i) {
            return (kon && s.count[i] >= k) || (!kon && fl.top_p < 1.0f && s.count[i] > 0 && s.mass[i] >= target) ||
                   (!(kon && fl.top_p < 1.0f) && fl.min_p > 0.0f && s.factor[i] < least);
        });
        if (s.count[b] <= kFew) {
            pick_few(row, s, b, s.count[b], fl, kon, whole, a.uniform[r], a.ids + r);
            return;
        }
    }
    // top-k, top-p, min-p, each narrowing what the one before has left; at most
    // one place in the buckets to resolve each (one loop, so that the code of it
    // is there once: a row's kernel runs through its code a single time)
    const double p = (double)fl.top_p;
    const double mp = fmin((double)fl.min_p, 1.0);
#pragma unroll 1
    for (int stage = 0; stage < 3; ++stage) {
        int b0 = 0, b1 = 0;
        long long take = 0;
        double target = 0.0;
        if (stage == 0) {
            if (!(k > 0 && k < tokens)) continue;
            b0 = b1 = first_bucket(s, [&](int i) { return s.count[i] >= k; });
            take = k - count_before(b0);
            if (take == s.count[b0] - count_before(b0)) {
                cut.bucket = b0;
                full = b0 + 1;
                kept = s.mass[b0];
                continue;
            }
        } else if (stage == 1) {
            if (!(p < 1.0)) continue;
            target = p > 0.0 ? p * kept - kSame * kept : 0.0;
            b0 = first_bucket(s, [&](int i) { return s.count[i] > 0 && s.mass[i] >= target; });
            if (b0 > cut.bucket) b0 = cut.bucket;
            b1 = b0;
        } else {
            if (!(mp > 0.0)) continue;
            // buckets that are neither whole above min_p nor whole below it
            b0 = first_bucket(s, [&](int i) { return s.factor[i] * 0.969233234476344 < mp * (1.0 + 1e-9); });  // e^(-1/32)
            b1 = first_bucket(s, [&](int i) { return s.factor[i] < mp * (1.0 - 1e-9); });
            if (b1 > b0) --b1;
            if (b1 > cut.bucket) b1 = cut.bucket;
            if (b0 > b1) continue;
            long long mine = 0, got, all;
            row.each(s, b0, b1, cut, [&](float l, uint32_t, int) { mine += 0x100000000ll + (row.weight(l) >= mp); });
            (void)block_scan<long long>(mine, s.wave_i, &all);
            got = all & 0xffffffffll;
            all >>= 32;
            if (got == 0 && b0 > 0) {
                cut.bucket = b0 - 1;
                full = b0;
                kept = mass_before(b0);
                continue;
            }
            if (got == all) {
                if (b1 < cut.bucket) {
                    cut.bucket = b1;
                    full = b1 + 1;
                    kept = mass_before(b1 + 1);
                }
                continue;
            }
            take = got;
        }
        kept = resolve(row, s, b0, b1, s.count[b1] - count_before(b0), take, target, mass_before(b0), &cut);
        full = b0;
    }

    // the segment where the kept mass passes u of the whole
    for (int i = wave; i < a.segs; i += kThreads / 64) {
        const int shift = s.shift[i];
        double m = 0.0;
#pragma unroll 8
        for (int j = 0; j < kBuckets / 64; ++j) {
            const int d = j * 64 + lane;  // of the row
            const bool in = d >= shift && d < full;
            const unsigned long long h = in ? row.hist[(long)i * kBuckets + d - shift] : 0;
            m += in ? ((double)(h >> 48) - (double)(h & kDefMask) * (1.0 / kDefUnit)) * s.factor[d] : 0.0;
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) m += __shfl_xor(m, d, 64);
        if (lane == 0) s.seg_mass[i] = m + (full <= cut.bucket ? (double)s.part[i] * (1.0 / kMassUnit) : 0.0);
    }
    __syncthreads();
    const double u = (double)a.uniform[r];
    const double goal = u > 0.0 ? u * kept + kSame * kept : 0.0;
    double total;
    double acc = block_scan<double>(tid < a.segs ? s.seg_mass[tid] : 0.0, s.wave_d, &total);
    if (tid == 0) s.found_j = kMaxSegs, s.found_i = 0;
    __syncthreads();
    if (tid < a.segs && s.seg_mass[tid] > 0.0) {
        if (acc > goal) atomicMin(&s.found_j, tid);
        atomicMax(&s.found_i, tid);
    }
    __syncthreads();
    const int seg = s.found_j < kMaxSegs ? s.found_j : s.found_i;
    if (tid == seg) s.found_mass = acc - s.seg_mass[tid];
    __syncthreads();
    const double want = goal - s.found_mass;
    __syncthreads();

    // and the token in it
    double w[8], sum = 0.0;
    const int i0 = seg * kSeg + 8 * tid;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float4 v = load4(row.x, a.vocab, i0 + 4 * j, a.vec);
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float l = usable(e[i]);
            double y = 0.0;
            if (l > -__builtin_inff()) {
                const uint32_t key = key_of(l);
                const int d = row.bucket(l);
                if (d <= cut.bucket && d < kBuckets &&
                    (key > cut.key || (key == cut.key && i0 + 4 * j + i <= cut.index))) {
                    y = row.weight(l);
                }
            }
            w[4 * j + i] = y;
            sum += y;
        }
    }
    acc = block_scan<double>(sum, s.wave_d, &total);
    if (tid == 0) s.found_j = kThreads, s.found_i = 0;
    __syncthreads();
    if (sum > 0.0) {
        if (acc > want) atomicMin(&s.found_j, tid);
        atomicMax(&s.found_i, tid);
    }
    __syncthreads();
    if (tid == (s.found_j < kThreads ? s.found_j : s.found_i)) {
        double upto = acc - sum;
        int id = at;
        for (int i = 0; i < 8; ++i) {
            if (w[i] <= 0.0) continue;
            upto += w[i];
            id = i0 + i;
            if (upto > want) break;
        }
        a.ids[r] = id;
    }
}

struct SampleLayout {
    size_t max, hist, first, list, bytes;
};

static SampleLayout sample_layout(int vocab, int rows) {
    const size_t n = (size_t)rows * ceil_div(vocab, kSeg);
    auto pad = [](size_t b) { return (b + 255) & ~(size_t)255; };
    SampleLayout l;
    l.max = 0;
    l.hist = pad(n * sizeof(SegMax));
    l.first = l.hist + n * kBuckets * 8;
    l.list = l.first + n * kBuckets * 2;
    l.bytes = l.list + n * kSeg * 2;
    return l;
}

size_t sample_workspace(int vocab, int rows) { return sample_layout(vocab, rows).bytes; }

hipError_t launch_sample(const SampleArgs& g, hipStream_t s) {
    SampleParams a;
    a.logits = g.logits;
    a.stride = g.stride;
    a.vocab = g.vocab;
    a.segs = ceil_div(g.vocab, kSeg);
    a.vec = ((uintptr_t)g.logits & 15) == 0 && g.stride % 4 == 0;
    a.temperature = g.temperature;
    a.top_k = g.top_k;
    a.top_p = g.top_p;
    a.min_p = g.min_p;
    a.uniform = g.uniform;
    a.ids = g.ids;
    const SampleLayout l = sample_layout(g.vocab, g.rows);
    char* w = (char*)g.workspace;
    a.seg_max = (SegMax*)(w + l.max);
    a.hist = (unsigned long long*)(w + l.hist);
    a.first = (uint16_t*)(w + l.first);
    a.list = (uint16_t*)(w + l.list);
    hipLaunchKernelGGL(sample_segments_kernel, dim3((unsigned)g.rows, (unsigned)a.segs), dim3(kThreads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_pick_kernel, dim3((unsigned)g.rows), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace lamd
