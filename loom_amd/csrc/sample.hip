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
constexpr double kFar = 0x1p30;  // |max / T| from which neighbouring floats are over 32 nats apart
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
    if (x != x) return -__builtin_inff();
    return fminf(x, 3.402823466e38f) + 0.0f;  // (-0 becomes +0)
}

// Order of values as unsigned integers.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

struct Better {
    __device__ __forceinline__ static bool before(float a, int ia, float b, int ib) {
        return a > b || (a == b && ia < ib);
    }
};

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

// z = l / T as a pair, and its bucket on the absolute grid of 1/32 nats.
struct Place {
    double z, lo, b;
};

__device__ __forceinline__ Place place(float l, double inv_t) {
    Place p;
    p.z = (double)l * inv_t;
    p.lo = __builtin_fma((double)l, inv_t, -p.z);
    p.b = floor(p.z * kPerNat);
    return p;
}

// Bucket of l under a largest value's (at distance d from it, or kBuckets when
// it is too far to have a mass).
__device__ __forceinline__ int bucket_of(const Place& p, const Place& top) {
    const double d = top.b - p.b;
    if (fabs(top.z) >= kFar) return p.z == top.z ? 0 : kBuckets;
    return d < (double)kBuckets ? (int)d : kBuckets;
}

// 1 - exp(r) for r in [-1/32, 0] (Taylor; the first term left out is 6e-15).
__device__ __forceinline__ double deficit(double r) {
    double y = 1.0 / 720.0;
    y = __builtin_fma(y, r, 1.0 / 120.0);
    y = __builtin_fma(y, r, 1.0 / 24.0);
    y = __builtin_fma(y, r, 1.0 / 6.0);
    y = __builtin_fma(y, r, 0.5);
    y = __builtin_fma(y, r, 1.0);
    return -r * y;
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

// Inclusive sums over the workgroup in thread order, and their total.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* wave_sum, T* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) wave_sum[wave] = v;
    __syncthreads();
    T before = 0, all = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
        const T x = wave_sum[w];
        if (w < wave) before += x;
        all += x;
    }
    *total = all;
    return v + before;
}

// One workgroup per (segment, row): its largest value, its histogram relative
// to it, and (where a filter may ask) its tokens listed by bucket.  A bucket's
// mass is kept as count and sum of 1 - exp(distance to the bucket's upper
// edge), one 64-bit LDS atomic a token, which is exact in any order and needs
// the row's maximum only when segments are joined; the atomic's old count is
// the token's place in its bucket's list.
__global__ __launch_bounds__(kThreads) void sample_segments_kernel(SampleParams a) {
    __shared__ unsigned long long hist[kBuckets];
    __shared__ uint16_t first[kBuckets];
    __shared__ __align__(16) uint16_t list[kSeg];
    __shared__ float sv[kThreads / 64];
    __shared__ int si[kThreads / 64];
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
    float best = -__builtin_inff();
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int idx = seg * kSeg + 4 * tid + (i >> 2) * 4 * kThreads + (i & 3);
        if (l[i] > best) best = l[i], at = idx;
    }
    block_best(best, at, sv, si);
    const long slot = row * a.segs + seg;
    if (!(fl.temperature > 0.0f) || best == -__builtin_inff()) {  // greedy, or nothing to draw: the maximum is all
        if (tid == 0) a.seg_max[slot] = SegMax{best, at, 0};
        return;
    }
    const double inv_t = 1.0 / (double)fl.temperature;
    const Place top = place(best, inv_t);
    const bool far = fabs(top.z) >= kFar;
    int place_of[8];  // bucket << 16 | place in it
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        place_of[i] = -1;
        if (l[i] == -__builtin_inff()) continue;
        const Place p = place(l[i], inv_t);
        const int d = bucket_of(p, top);
        if (d >= kBuckets) continue;
        double r = far ? 0.0 : (p.z - (p.b + 1.0) / kPerNat) + p.lo;
        r = fmin(fmax(r, -1.0 / kPerNat), 0.0);
        const unsigned long long old = atomicAdd(&hist[d], (1ull << 48) | (unsigned long long)(deficit(r) * kDefUnit + 0.5));
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
    if (tid == 0) a.seg_max[slot] = SegMax{best, at, listed};
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
    double inv_t;
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
    __device__ __forceinline__ int bucket(float l) const { return bucket_of(place(l, inv_t), top); }

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

// One workgroup per row.
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
    row.top = place(best, row.inv_t);
    row.seg_max = sm;
    row.hist = a.hist + r * a.segs * kBuckets;
    row.first = a.first + r * a.segs * kBuckets;
    row.list = a.list + r * a.segs * kSeg;
    const bool far = fabs(row.top.z) >= kFar;

    // the segments' histograms on the row's grid
    for (int i = tid; i < a.segs; i += kThreads) {
        const float v = sm[i].value;
        s.shift[i] = v == -__builtin_inff() ? kBuckets : bucket_of(place(v, row.inv_t), row.top);
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
    const double edge = far ? (tid == 0 ? 0.0 : -1e30) : ((row.top.b - tid + 1.0) / kPerNat - row.top.z) - row.top.lo;
    const double factor = exp(edge);
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
    if (k > 0 && k < tokens) {
        const int b = first_bucket(s, [&](int i) { return s.count[i] >= k; });
        const long long nb = s.count[b] - count_before(b), take = k - count_before(b);
        if (take == nb) {
            cut.bucket = b;
            full = b + 1;
            kept = s.mass[b];
        } else {
            kept = resolve(row, s, b, b, nb, take, 0.0, mass_before(b), &cut);
            full = b;
        }
    }
    const double p = (double)fl.top_p;
    if (p < 1.0) {
        const double target = p > 0.0 ? p * kept - kSame * kept : 0.0;
        int b = first_bucket(s, [&](int i) { return s.count[i] > 0 && s.mass[i] >= target; });
        if (b > cut.bucket) b = cut.bucket;
        const long long nb = s.count[b] - count_before(b);
        kept = resolve(row, s, b, b, nb, 0, target, mass_before(b), &cut);
        full = b;
    }
    double mp = (double)fl.min_p;
    if (mp > 1.0) mp = 1.0;
    if (mp > 0.0) {
        // buckets that are neither whole above min_p nor whole below it
        const int b0 = first_bucket(s, [&](int i) { return s.factor[i] * exp(-1.0 / kPerNat) < mp * (1.0 + 1e-9); });
        int b1 = first_bucket(s, [&](int i) { return s.factor[i] < mp * (1.0 - 1e-9); });
        if (b1 > b0) --b1;
        if (b1 > cut.bucket) b1 = cut.bucket;
        if (b0 <= b1) {
            int mine = 0, of = 0;
            row.each(s, b0, b1, cut, [&](float l, uint32_t, int) {
                ++of;
                mine += row.weight(l) >= mp;
            });
            long long got, all;
            (void)block_scan<long long>(mine, s.wave_i, &got);
            (void)block_scan<long long>(of, s.wave_i, &all);
            if (got == 0 && b0 > 0) {
                cut.bucket = b0 - 1;
                full = b0;
                kept = mass_before(b0);
            } else if (got == all) {
                if (b1 < cut.bucket) {
                    cut.bucket = b1;
                    full = b1 + 1;
                    kept = mass_before(b1 + 1);
                }
            } else {
                kept = resolve(row, s, b0, b1, s.count[b1] - count_before(b0), got, 0.0, mass_before(b0), &cut);
                full = b0;
            }
        }
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
