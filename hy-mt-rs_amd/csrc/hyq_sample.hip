// Tokens drawn from rows of logits with temperature, top-k, top-p and min-p
// and a given random number u in [0, 1).
//
//   w_i = exp((l_i - max l) / T)
//   order: larger l first, equal ones by index
//   kept: the first k of the order; of those the shortest prefix whose weight
//   reaches top_p of their weight; of those the ones with w_i >= min_p
//   token: in index order the first kept i with w_0 + .. + w_i > u * W
//
// Every filter keeps a prefix of the order, so the kept set is one cut: a
// value, and for equal values an index. Weights are formed in 64 bits and held
// as integers w_i 2^shift, so that their sums are exact and do not depend on
// the order of addition: sums by any number of workgroups give the same bits
// always, and a border falls where 64-bit arithmetic puts it. Weights below
// e^-32 of the largest are zero and never drawn (shift is 62 minus log2 of the
// vocabulary, at most 46; e^-32 = 2^-46.2).
//
// A row is cut into splits of a workgroup each, over three launches that each
// read the row once, and a last one with a workgroup per row:
//   max     the largest value and its first index, by split
//   bins    a histogram, by split, of (max - l) / T in 2048 bins of 1/64:
//           counts where top-k is set, weights where top-p needs them
//   sums    every workgroup adds the splits' histograms and finds the bins that
//           the cuts fall into; their members go to a list, and the weights of
//           all smaller bins are summed by split
//   draw    sorts the list, cuts it exactly, adds the kept members to the
//           splits' sums, finds the split that holds u W and in it the token
// Where a cut's bin has more members than the list holds (equal logits by the
// thousand) the last launch does the row by itself, refining its cut bit by
// bit over the row.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef unsigned long long u64;

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_WAVES = SAMPLE_THREADS / 64;
constexpr int SAMPLE_BINS = 2048;  // 1/64 wide: 32 in all
constexpr int SAMPLE_LIST = 2048;  // members of a cut's bins
constexpr int SAMPLE_SMALL = 1024; // the largest top-k whose members are listed whole
constexpr int SAMPLE_SPLITS = 32;

// An integer that orders floats (a NaN as minus infinity).
__device__ __forceinline__ unsigned order_key(float x)
{
    if (x != x) x = -INFINITY;
    if (x == 0.f) x = 0.f; // the two zeros are equal
    const unsigned b = __builtin_bit_cast(unsigned, x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

struct RowSettings {
    float max, per_bin; // 64 / T
    double inv_t, scale, min_p;
};
// The bin of a value, SAMPLE_BINS where its weight is zero. (Rounding is
// monotone, so larger values never have larger bins.)
__device__ __forceinline__ int bin_of(float l, const RowSettings &s)
{
    if (l == s.max) return 0;
    const float d = (s.max - l) * s.per_bin; // (NaN and infinite: no bin)
    return d < (float)SAMPLE_BINS ? (int)d : SAMPLE_BINS;
}
// exp(x) for x in [-33, 0]: x = n ln 2 + r with |r| <= 0.347, the series of
// exp(r) to r^12 (the next term is below 2e-16), times 2^n.
__device__ __forceinline__ double exp_neg(double x)
{
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));
    double e = 1.0 / 479001600;
    e = fma(e, r, 1.0 / 39916800);
    e = fma(e, r, 1.0 / 3628800);
    e = fma(e, r, 1.0 / 362880);
    e = fma(e, r, 1.0 / 40320);
    e = fma(e, r, 1.0 / 5040);
    e = fma(e, r, 1.0 / 720);
    e = fma(e, r, 1.0 / 120);
    e = fma(e, r, 1.0 / 24);
    e = fma(e, r, 1.0 / 6);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    return ldexp(e, (int)n);
}
// The weight of a value that has a bin.
__device__ __forceinline__ double weight(float l, const RowSettings &s)
{
    if (l == s.max) return 1.0;
    return exp_neg(((double)l - (double)s.max) * s.inv_t);
}
__device__ __forceinline__ u64 fixed(double w, const RowSettings &s)
{
    return (u64)(w * s.scale + 0.5);
}

__device__ __forceinline__ u64 wave_sum(u64 v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v, int lane) // inclusive
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}

// Inclusive scan over the workgroup; *all is the total.
__device__ __forceinline__ u64 block_scan(u64 v, u64 *wsum, u64 *all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    u64 base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < SAMPLE_WAVES; ++w) {
        if (w < wave) base += wsum[w];
        sum += wsum[w];
    }
    *all = sum;
    return base + v;
}

struct Cut {
    unsigned key; // kept: a larger key, or this one and an index <= last
    int last;
};

struct SampleArgs {
    const float *logits;
    int vocab, shift, splits, per; // per: values of a split
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *random;
    int *token;
    float *prob;
    // scratch
    float *smax;     // [rows][splits]
    int *sidx;       // [rows][splits]: the split's first maximum
    unsigned *count; // [rows][splits][SAMPLE_BINS]
    u64 *wsum;       // [rows][splits][SAMPLE_BINS]
    u64 *sums;       // [rows][splits]: weights of the bins before the listed ones
    struct Found *found; // [rows]
    unsigned *have;  // [rows][2]: members listed
    u64 *list;       // [rows][2][SAMPLE_LIST]: order key << 32 | ~index
};

// What the histogram says of a row's cuts. List 0 takes the bins lo .. hi, in
// which the kept set ends; list 1 the bin kbin, where it is not among those
// and the top-k's own cut is needed first, for the weight that top-p is of.
struct Found {
    int lo, hi, kbin;         // (kbin -1: no list 1)
    int k_in_list;            // the top-k's cut, if it cuts, lies in list 0
    unsigned before, kbefore; // counts of the bins before lo, and before kbin
    u64 wbefore, kwbefore;    // and weights (lo: where top-p cuts)
    u64 total;                // the weight of all bins, where top-p cuts
};

struct RowPlan {
    bool greedy;        // no weights: the first maximum, or nothing
    bool by_k, by_p;    // which filters cut
    bool counts, sums;  // which histograms they need
    float max;
    int first;          // index of the first maximum
    int k;
    double p;
    RowSettings st;
};

// The row's maximum from its splits' and its settings. Uniform.
__device__ __forceinline__ RowPlan plan_row(const SampleArgs &a, int row)
{
    static_assert(SAMPLE_SPLITS <= 64, "a split per lane");
    RowPlan r;
    const int lane = threadIdx.x & 63, at = row * a.splits + min(lane, a.splits - 1);
    const float m = a.smax[at];
    const int idx = a.sidx[at];
    r.max = wave::max64(m);
    // (splits ascend: the first lane of the maximum has its first index)
    r.first = __builtin_amdgcn_readlane(idx, __ffsll((long long)__ballot(m == r.max)) - 1);
    const float temp = a.temperature[row];
    r.greedy = !(r.max > -INFINITY) || !(temp > 0.f);
    r.k = a.top_k[row];
    r.p = a.top_p[row];
    r.by_k = r.k > 0 && r.k < a.vocab;
    r.by_p = r.p < 1.0;
    // a small top-k's members are listed whole, and need no weights before
    r.counts = !r.greedy && r.by_k;
    r.sums = !r.greedy && r.by_p && !(r.by_k && r.k <= SAMPLE_SMALL);
    r.st.max = r.max;
    r.st.inv_t = 1.0 / (double)temp;
    r.st.per_bin = (float)(64.0 * r.st.inv_t);
    r.st.scale = ldexp(1.0, a.shift);
    const float least = a.min_p[row];
    r.st.min_p = least > 0.f ? fmin((double)least, 1.0) : 0.0;
    return r;
}

// The prefix weight that top-p asks for, of `total`.
__device__ __forceinline__ u64 top_p_target(double p, u64 total)
{
    const double want = fmax(p, 0.0) * (double)total;
    u64 target = (u64)want;
    if ((double)target < want) ++target;
    return min(max(target, (u64)1), total);
}
// The first running weight that exceeds u W is the first to reach this.
__device__ __forceinline__ u64 draw_target(float random, u64 total)
{
    const double u = fmin(fmax((double)random, 0.0), 1.0);
    return min((u64)(u * (double)total) + 1, total);
}

// ---- max ----
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_max_kernel(SampleArgs a)
{
    __shared__ float sm[SAMPLE_WAVES];
    __shared__ int si[SAMPLE_WAVES];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const float *x = a.logits + (size_t)row * a.vocab;
    const int end = min(a.vocab, (s + 1) * a.per);
    float mx = -INFINITY;
    int mi = 0x7fffffff;
    for (int i = s * a.per + t; i < end; i += 4 * SAMPLE_THREADS) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = x[min(i + u * SAMPLE_THREADS, end - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * SAMPLE_THREADS < end && v[u] > mx) {
                mx = v[u];
                mi = i + u * SAMPLE_THREADS;
            }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float v = __shfl_xor(mx, o, 64);
        const int i = __shfl_xor(mi, o, 64);
        if (v > mx || (v == mx && i < mi)) {
            mx = v;
            mi = i;
        }
    }
    if ((t & 63) == 0) {
        sm[t >> 6] = mx;
        si[t >> 6] = mi;
    }
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < SAMPLE_WAVES; ++w)
            if (sm[w] > mx || (sm[w] == mx && si[w] < mi)) {
                mx = sm[w];
                mi = si[w];
            }
        a.smax[row * a.splits + s] = mx;
        a.sidx[row * a.splits + s] = mi;
        if (s == 0) a.have[2 * row] = a.have[2 * row + 1] = 0;
    }
}

// ---- bins ----
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_bins_kernel(SampleArgs a)
{
    __shared__ u64 hw[SAMPLE_BINS];
    __shared__ unsigned hc[SAMPLE_BINS];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const RowPlan r = plan_row(a, row);
    if (!r.counts && !r.sums) return;
    const float *x = a.logits + (size_t)row * a.vocab;
    const int end = min(a.vocab, (s + 1) * a.per);
    for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
        hw[b] = 0;
        hc[b] = 0;
    }
    __syncthreads();
    for (int i = s * a.per + t; i < end; i += 4 * SAMPLE_THREADS) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = x[min(i + u * SAMPLE_THREADS, end - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int b = bin_of(v[u], r.st);
            if (i + u * SAMPLE_THREADS >= end || b >= SAMPLE_BINS) continue;
            if (r.counts) atomicAdd(hc + b, 1u);
            if (r.sums) atomicAdd(hw + b, fixed(weight(v[u], r.st), r.st));
        }
    }
    __syncthreads();
    const size_t at = ((size_t)row * a.splits + s) * SAMPLE_BINS;
    for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
        if (r.counts) a.count[at + b] = hc[b];
        if (r.sums) a.wsum[at + b] = hw[b];
    }
}

// ---- sums ----
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_sums_kernel(SampleArgs a)
{
    __shared__ u64 wsum[SAMPLE_WAVES];
    __shared__ Found f;
    __shared__ unsigned listed[2], base[2];
    __shared__ u64 list[2][SAMPLE_LIST];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const RowPlan r = plan_row(a, row);
    if (r.greedy) return;
    if (t == 0) {
        f = Found{SAMPLE_BINS, SAMPLE_BINS, -1, 0, 0, 0, 0, 0, 0}; // nothing cut: all bins summed
        listed[0] = listed[1] = 0;
    }
    if (r.counts || r.sums) {
        // this thread's two bins over all splits, and their running totals
        u64 c0 = 0, c1 = 0, w0 = 0, w1 = 0, ctotal = 0, wtotal = 0;
        const size_t at = (size_t)row * a.splits * SAMPLE_BINS + 2 * t;
#pragma unroll 8
        for (int i = 0; i < a.splits; ++i) {
            if (r.counts) {
                const uint2 c =
                    *reinterpret_cast<const uint2 *>(a.count + at + (size_t)i * SAMPLE_BINS);
                c0 += c.x;
                c1 += c.y;
            }
            if (r.sums) {
                const ulonglong2 w =
                    *reinterpret_cast<const ulonglong2 *>(a.wsum + at + (size_t)i * SAMPLE_BINS);
                w0 += w.x;
                w1 += w.y;
            }
        }
        const u64 cup = block_scan(c0 + c1, wsum, &ctotal);
        const u64 wup = block_scan(w0 + w1, wsum, &wtotal);
        const u64 cb = cup - c0 - c1, wb = wup - w0 - w1;
        // which of this thread's bins a running value reaches a target in: -1, 0, 1
        auto reaches = [](u64 before, u64 x0, u64 x1, u64 target) {
            return before < target && before + x0 + x1 >= target ? (before + x0 < target) : -1;
        };
        const bool cuts = r.by_k && (u64)r.k < ctotal;
        if (cuts) {
            const int i = reaches(cb, c0, c1, r.k);
            if (i >= 0) {
                f.kbin = 2 * t + i;
                f.kbefore = (unsigned)(i ? cb + c0 : cb);
                f.kwbefore = i ? wb + w0 : wb;
                f.hi = i ? 1 : 0; // (for now: which of the thread's bins)
                f.total = (i ? wb + w0 + w1 : wb + w0); // the weight through kbin
            }
        }
        __syncthreads();
        const bool small = r.by_k && r.k <= SAMPLE_SMALL;
        const u64 least = cuts ? f.kwbefore : wtotal, most = cuts ? f.total : wtotal;
        __syncthreads();
        if (small) {
            // the order's first k and top-p in them: all in the list
            if (t == 0) {
                f.lo = 0;
                f.hi = cuts ? f.kbin : SAMPLE_BINS - 1;
                f.kbin = -1;
                f.k_in_list = 1;
            }
        } else if (r.by_p) {
            // top-p of a weight between least and most
            const int i = reaches(wb, w0, w1, top_p_target(r.p, max(least, (u64)1)));
            const int j = reaches(wb, w0, w1, top_p_target(r.p, max(most, (u64)1)));
            if (i >= 0) {
                f.lo = 2 * t + i;
                f.before = (unsigned)(i ? cb + c0 : cb);
                f.wbefore = i ? wb + w0 : wb;
            }
            if (j >= 0) f.hi = 2 * t + j;
            if (t == 0) f.total = wtotal;
        } else if (cuts && t == 0) {
            f.lo = f.hi = f.kbin;
            f.before = f.kbefore;
            f.kbin = -1;
            f.k_in_list = 1;
        } else if (t == 0) {
            f.lo = f.hi = SAMPLE_BINS;
        }
        __syncthreads();
        if (t == 0 && f.kbin >= 0 && f.kbin <= f.hi) { // (in list 0 already)
            f.hi = f.kbin;
            f.kbin = -1;
            f.k_in_list = 1;
        }
    }
    __syncthreads();
    const Found g = f;
    if (s == 0 && t == 0) a.found[row] = g;

    const float *x = a.logits + (size_t)row * a.vocab;
    const int end = min(a.vocab, (s + 1) * a.per);
    u64 sum = 0;
    for (int i = s * a.per + t; i < end; i += 4 * SAMPLE_THREADS) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = x[min(i + u * SAMPLE_THREADS, end - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = i + u * SAMPLE_THREADS, b = bin_of(v[u], r.st);
            if (j >= end || b >= SAMPLE_BINS) continue;
            if (b < g.lo) {
                const double w = weight(v[u], r.st);
                if (w >= r.st.min_p) sum += fixed(w, r.st);
            }
            const int which = b >= g.lo && b <= g.hi ? 0 : b == g.kbin ? 1 : -1;
            if (which >= 0) {
                const unsigned n = atomicAdd(listed + which, 1u);
                if (n < SAMPLE_LIST)
                    list[which][n] = (u64)order_key(v[u]) << 32 | (unsigned)~j;
            }
        }
    }
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) wsum[wave] = sum;
    if (t < 2) base[t] = listed[t] ? atomicAdd(a.have + 2 * row + t, listed[t]) : 0;
    __syncthreads();
    if (t == 0) {
        u64 all = 0;
        for (int w = 0; w < SAMPLE_WAVES; ++w) all += wsum[w];
        a.sums[row * a.splits + s] = all;
    }
    for (int which = 0; which < 2; ++which)
        for (unsigned n = t; n < min(listed[which], (unsigned)SAMPLE_LIST); n += SAMPLE_THREADS)
            if (base[which] + n < SAMPLE_LIST)
                a.list[((size_t)row * 2 + which) * SAMPLE_LIST + base[which] + n] = list[which][n];
}

// ---- draw ----
// Sorts n <= SAMPLE_LIST keys in LDS, largest first.
__device__ __forceinline__ void sort_desc(u64 *key, int n)
{
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += SAMPLE_THREADS) key[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int e = threadIdx.x; e < size / 2; e += SAMPLE_THREADS) {
                const int lo = 2 * e - (e & (j - 1)), hi = lo + j;
                const u64 x = key[lo], y = key[hi];
                if ((x < y) == ((lo & k) == 0)) {
                    key[lo] = y;
                    key[hi] = x;
                }
            }
            __syncthreads();
        }
}

__device__ __forceinline__ float value_of(u64 key) // the float of an order key
{
    const unsigned k = (unsigned)(key >> 32);
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The whole row by one workgroup (see the head of the file).
__device__ __noinline__ void row_alone(const SampleArgs &a, const RowPlan &plan, int row,
                                       u64 *hw, unsigned *hc, u64 *wsum, u64 *pick)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, vocab = a.vocab, k = plan.k;
    const float *x = a.logits + (size_t)row * vocab;
    const double p = plan.p;
    const RowSettings st = plan.st;
    for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
        hw[b] = 0;
        hc[b] = 0;
    }
    __syncthreads();
    for (int i = t; i < vocab; i += SAMPLE_THREADS) {
        const float v = x[i];
        const int b = bin_of(v, st);
        if (b < SAMPLE_BINS) {
            atomicAdd(hc + b, 1u);
            atomicAdd(hw + b, fixed(weight(v, st), st));
        }
    }
    __syncthreads();
    // a scan of the two bins of each thread
    u64 total, count;
    const u64 w0 = hw[2 * t], w1 = hw[2 * t + 1];
    const u64 c0 = hc[2 * t], c1 = hc[2 * t + 1];
    const u64 wup = block_scan(w0 + w1, wsum, &total);
    const u64 cup = block_scan(c0 + c1, wsum, &count);

    Cut cut = {0, 0x7fffffff};
    // Cuts the order inside bin b so that the prefix has `target` (counts, or
    // weight when `byw`), of which `before` lies in smaller bins. Returns the
    // weight of the prefix from `wbefore`, that of the smaller bins.
    auto resolve = [&](int b, u64 target, u64 before, u64 wbefore, bool byw) {
        unsigned prefix = 0;
        for (int level = 0; level < 4; ++level) {
            const int sh = 24 - 8 * level;
            __syncthreads();
            if (t < 256) {
                hw[t] = 0;
                hc[t] = 0;
            }
            __syncthreads();
            for (int i = t; i < vocab; i += SAMPLE_THREADS) {
                const float v = x[i];
                const unsigned key = order_key(v);
                if (level && (key >> (sh + 8)) != prefix) continue;
                if (bin_of(v, st) != b) continue;
                atomicAdd(hc + ((key >> sh) & 255), 1u);
                atomicAdd(hw + ((key >> sh) & 255), fixed(weight(v, st), st));
            }
            __syncthreads();
            if (t == 0) {
                int d = 255;
                u64 a = before, wa = wbefore;
                for (; d > 0; --d) {
                    const u64 add = byw ? hw[d] : hc[d];
                    if (a + add >= target) break;
                    a += add;
                    wa += hw[d];
                }
                pick[0] = d;
                pick[1] = a;
                pick[2] = wa;
                pick[3] = hc[d] ? hw[d] / hc[d] : 0; // at the last level: one value's weight
            }
            __syncthreads();
            prefix = prefix << 8 | (unsigned)pick[0];
            before = pick[1];
            wbefore = pick[2];
        }
        const u64 each = pick[3];
        // (values whose weight rounds to zero add nothing: the first will do)
        const u64 ties = !byw ? target - before : each ? (target - before + each - 1) / each : 1;
        // the index of the last of the first `ties` equal values
        cut.key = prefix;
        const int per = (vocab + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
        const int i0 = min(vocab, t * per), i1 = min(vocab, i0 + per);
        u64 mine = 0, all;
        for (int i = i0; i < i1; ++i) mine += order_key(x[i]) == prefix;
        const u64 upto = block_scan(mine, wsum, &all);
        if (mine && upto >= ties && upto - mine < ties) {
            u64 a = upto - mine;
            for (int i = i0; i < i1; ++i)
                if (order_key(x[i]) == prefix && ++a == ties) {
                    pick[0] = i;
                    break;
                }
        }
        __syncthreads();
        cut.last = (int)pick[0];
        return wbefore + ties * each;
    };
    // the bin where the running value (inclusive `up` after this thread's two
    // bins a0, a1) reaches target: bin, value before it
    auto find = [&](u64 up, u64 a0, u64 a1, u64 other, u64 o0, u64 o1, u64 target) {
        __syncthreads();
        const u64 base = up - a0 - a1, obase = other - o0 - o1;
        if (up >= target && base < target) {
            const bool second = base + a0 < target;
            pick[0] = 2 * t + second;
            pick[1] = second ? base + a0 : base;
            pick[2] = second ? obase + o0 : obase;
        }
        __syncthreads();
    };
    if (k > 0 && (u64)k < count) {
        find(cup, c0, c1, wup, w0, w1, k);
        const int b = (int)pick[0];
        const u64 before = pick[1], wbefore = pick[2];
        total = resolve(b, k, before, wbefore, false);
    }
    if (p < 1.0) {
        const u64 target = top_p_target(p, total);
        find(wup, w0, w1, wup, w0, w1, target);
        const int b = (int)pick[0];
        const u64 before = pick[1];
        resolve(b, target, before, before, true);
    }

    // the kept weights in index order: sums of each wave's range, then of 16
    // parts of the range that holds the target, then one by one
    auto kept = [&](int i) -> u64 {
        const float v = x[i];
        const unsigned key = order_key(v);
        if (key < cut.key || (key == cut.key && i > cut.last)) return 0;
        if (bin_of(v, st) >= SAMPLE_BINS) return 0;
        const double w = weight(v, st);
        return w >= st.min_p ? fixed(w, st) : 0;
    };
    int lo = 0, hi = vocab;
    u64 before = 0, target = 0, whole = 0;
    for (int level = 0; level < 2; ++level) {
        const int per = (hi - lo + SAMPLE_WAVES - 1) / SAMPLE_WAVES;
        const int i0 = min(hi, lo + wave * per), i1 = min(hi, i0 + per);
        u64 mine = 0;
        for (int i = i0 + lane; i < i1; i += 64) mine += kept(i);
        mine = wave_sum(mine);
        __syncthreads();
        if (lane == 0) wsum[wave] = mine;
        __syncthreads();
        if (level == 0) {
            for (int w = 0; w < SAMPLE_WAVES; ++w) whole += wsum[w];
            target = draw_target(a.random[row], whole);
        }
        int w = 0;
        for (; w < SAMPLE_WAVES - 1 && before + wsum[w] < target; ++w) before += wsum[w];
        lo = min(hi, lo + w * per);
        hi = min(hi, lo + per);
    }
    __syncthreads();
    if (wave == 0) {
        for (int b = lo; b < hi; b += 64) {
            const u64 w = b + lane < hi ? kept(b + lane) : 0;
            const u64 upto = before + wave_scan(w, lane);
            const u64 hit = __ballot(upto >= target);
            if (hit) {
                const int f = __ffsll((long long)hit) - 1;
                if (lane == f) {
                    a.token[row] = b + lane;
                    if (a.prob)
                        a.prob[row] =
                            (float)(weight(x[b + lane], st) * st.scale / (double)whole);
                }
                break;
            }
            before = __shfl(upto, 63, 64);
        }
    }
}


__global__ __launch_bounds__(SAMPLE_THREADS) void sample_draw_kernel(SampleArgs a)
{
    __shared__ u64 hw[SAMPLE_BINS];
    __shared__ unsigned hc[SAMPLE_BINS];
    __shared__ u64 wsum[SAMPLE_WAVES];
    __shared__ u64 pick[4];
    __shared__ u64 split_sum[SAMPLE_SPLITS];
    __shared__ u64 key[SAMPLE_LIST];
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const RowPlan r = plan_row(a, row);
    if (r.greedy) { // the first maximum, or nothing to take
        if (t == 0) {
            const bool any = r.max > -INFINITY;
            a.token[row] = any ? r.first : -1;
            if (a.prob) a.prob[row] = any ? 1.f : 0.f;
        }
        return;
    }
    const RowSettings &st = r.st;
    const Found f = a.found[row];
    const unsigned n0 = a.have[2 * row], n1 = a.have[2 * row + 1];
    if (n0 > SAMPLE_LIST || n1 > SAMPLE_LIST) {
        row_alone(a, r, row, hw, hc, wsum, pick);
        return;
    }
    const u64 *lists = a.list + (size_t)row * 2 * SAMPLE_LIST;
    // a thread's members 2 t and 2 t + 1 of a sorted list, and the running
    // weight before them
    auto load = [&](int which, int n) {
        for (int i = t; i < n; i += SAMPLE_THREADS) key[i] = lists[which * SAMPLE_LIST + i];
        __syncthreads();
        sort_desc(key, n);
    };
    auto weight_at = [&](int i, int n) -> u64 {
        return i < n ? fixed(weight(value_of(key[i]), st), st) : 0;
    };
    // the weight that top-p is of
    u64 of = f.total;
    if (f.kbin >= 0) {
        load(1, n1);
        const int n = min((int)n1, r.k - (int)f.kbefore);
        u64 all;
        block_scan(weight_at(2 * t, n) + weight_at(2 * t + 1, n), wsum, &all);
        of = f.kwbefore + all;
        __syncthreads();
    }
    // the members kept by top-k and top-p: the first `kept`
    int kept = (int)n0;
    u64 w0 = 0, w1 = 0;
    if (n0) {
        load(0, n0);
        if (f.k_in_list) kept = min(kept, r.k - (int)f.before);
        w0 = weight_at(2 * t, kept);
        w1 = weight_at(2 * t + 1, kept);
        if (r.by_p) {
            u64 all;
            const u64 up = block_scan(w0 + w1, wsum, &all);
            if (f.k_in_list) of = f.wbefore + all;
            const u64 target = top_p_target(r.p, max(of, (u64)1));
            const u64 b = f.wbefore + up - w0 - w1;
            if (t == 0) pick[0] = kept;
            __syncthreads();
            if (b < target && b + w0 + w1 >= target) pick[0] = 2 * t + (b + w0 < target ? 2 : 1);
            __syncthreads();
            kept = (int)pick[0];
        }
    }
    // the kept members' weights to their splits
    if (t < a.splits) split_sum[t] = a.sums[row * a.splits + t];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = 2 * t + i;
        if (j >= kept || (int)n0 <= j) continue;
        if (weight(value_of(key[j]), st) >= st.min_p)
            atomicAdd(split_sum + (int)(~(unsigned)key[j]) / a.per, i ? w1 : w0);
    }
    __syncthreads();
    // the split that holds the target, and the token in it
    const u64 mine_s = lane < a.splits ? split_sum[lane] : 0, upto_s = wave_scan(mine_s, lane);
    const u64 whole = __shfl(upto_s, 63, 64);
    const u64 target = draw_target(a.random[row], whole);
    const int s = min(__ffsll((long long)__ballot(upto_s >= target)) - 1, a.splits - 1);
    u64 before = __shfl(upto_s - mine_s, s, 64);
    const u64 last = n0 && kept ? key[kept - 1] : 0; // kept: this key and larger ones
    const float *x = a.logits + (size_t)row * a.vocab;
    auto kept_weight = [&](int i) -> u64 {
        const float v = x[i];
        const int b = bin_of(v, st);
        if (b >= SAMPLE_BINS || b > f.hi) return 0;
        if (b >= f.lo && (kept == 0 || ((u64)order_key(v) << 32 | (unsigned)~i) < last)) return 0;
        const double w = weight(v, st);
        return w >= st.min_p ? fixed(w, st) : 0;
    };
    const int begin = s * a.per, end = min(a.vocab, begin + a.per);
    // by runs of a wave: 64 consecutive values a step
    const int run = ((end - begin + SAMPLE_WAVES - 1) / SAMPLE_WAVES + 63) / 64 * 64;
    const int i0 = begin + wave * run, i1 = min(end, i0 + run);
    u64 mine = 0;
    for (int i = i0 + lane; i < i1; i += 64) mine += kept_weight(i);
    mine = wave_sum(mine);
    if (lane == 0) wsum[wave] = mine;
    __syncthreads();
    const u64 mine_w = lane < SAMPLE_WAVES ? wsum[lane] : 0;
    const u64 upto_w = before + wave_scan(mine_w, lane);
    const int w = __ffsll((long long)__ballot(upto_w >= target)) - 1;
    if (wave != w) return;
    before = __shfl(upto_w - mine_w, w, 64);
    for (int b = i0; b < i1; b += 64) {
        const u64 v = b + lane < i1 ? kept_weight(b + lane) : 0;
        const u64 upto = before + wave_scan(v, lane);
        const u64 hit = __ballot(upto >= target);
        if (hit) {
            const int at = __ffsll((long long)hit) - 1;
            if (lane == at) {
                a.token[row] = b + lane;
                if (a.prob)
                    a.prob[row] = (float)(weight(x[b + lane], st) * st.scale / (double)whole);
            }
            break;
        }
        before = __shfl(upto, 63, 64);
    }
}

struct SampleLayout {
    int splits, per;
    size_t sidx, count, wsum, sums, found, have, list, bytes;
};
// Splits: as many workgroups as fill the GPU twice, but at most 32 (each
// workgroup of the third launch adds up all of a row's histograms) and none of
// fewer than 1024 values.
SampleLayout sample_layout(int rows, int vocab)
{
    SampleLayout l;
    const int most = (vocab + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
    l.splits = std::max(1, std::min({512 / rows, SAMPLE_SPLITS, most}));
    l.per = (vocab + l.splits - 1) / l.splits;
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t n = (size_t)rows * l.splits;
    l.sidx = up(n * 4);
    l.count = l.sidx + up(n * 4);
    l.wsum = l.count + n * SAMPLE_BINS * 4;
    l.sums = l.wsum + n * SAMPLE_BINS * 8;
    l.found = l.sums + up(n * 8);
    l.have = l.found + up(rows * sizeof(Found));
    l.list = l.have + up((size_t)rows * 8);
    l.bytes = l.list + (size_t)rows * 2 * SAMPLE_LIST * 8;
    return l;
}

} // namespace

size_t sample_scratch(int rows, int vocab) { return sample_layout(rows, vocab).bytes; }

int launch_sample(const float *logits, int rows, int vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *random,
                  void *scratch, int *token, float *prob, void *stream)
{
    if (rows <= 0) return 0;
    int bits = 0;
    while ((1ll << bits) < vocab) ++bits;
    const SampleLayout l = sample_layout(rows, vocab);
    char *base = (char *)scratch;
    SampleArgs a{};
    a.logits = logits;
    a.vocab = vocab;
    a.shift = std::min(46, 62 - bits);
    a.splits = l.splits;
    a.per = l.per;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.random = random;
    a.token = token;
    a.prob = prob;
    a.smax = (float *)base;
    a.sidx = (int *)(base + l.sidx);
    a.count = (unsigned *)(base + l.count);
    a.wsum = (u64 *)(base + l.wsum);
    a.sums = (u64 *)(base + l.sums);
    a.found = (Found *)(base + l.found);
    a.have = (unsigned *)(base + l.have);
    a.list = (u64 *)(base + l.list);
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(l.splits, rows), block(SAMPLE_THREADS);
    hipLaunchKernelGGL(sample_max_kernel, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_bins_kernel, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_sums_kernel, grid, block, 0, st, a);
    hipLaunchKernelGGL(sample_draw_kernel, dim3(rows), block, 0, st, a);
    return (int)hipGetLastError();
}

} // namespace hyq
