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
// A row is cut into splits of a workgroup each, a split into a run per wave:
//   max     the largest value and its first index, by split
//   bins    a histogram, by split, of (max - l) / T in 2048 bins of 1/64:
//           counts where top-k is set, weights where top-p needs them
//   find    (a workgroup per row; of few rows, every workgroup of the next launch)
//           adds the splits' histograms and finds the bins that the cuts fall into
//   sums    lists those bins' members, and sums the weights of the smaller bins
//           by run
//   draw    (a workgroup per row) cuts the list exactly, adds the kept members
//           to the runs' sums, finds the run that holds u W and in it the token
// Where a cut's bin has more members than the list holds (equal logits by the
// thousand) the last launch does the row by itself, refining its cut bit by bit
// over the row: a dozen passes by one workgroup where both cuts fall among ties.
// Rows of 128167 equal logits with top-p take 1.3 ms, with top-k 50000 as well 2.3
// (64 of them 1.4 and 2.5); rounded to quarters 0.5 and 0.8.
//
// Two rows of 120818 with top-k 20 and top-p are four short launches, 20.7 us (2.6,
// 4.4, 9.2, 5.6). 64 rows of 128167 with settings of all kinds take 57 us:
// max 6 (the logits' stream), bins 13 and sums 16 (instructions, some 55 for each
// value weighed, of which ten are 64-bit operations), find 8 and draw 15 (a
// workgroup per row: latency).
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
constexpr int SAMPLE_SPLITS = 16;
// Up to this many rows the splits' workgroups find the cuts each for itself: 256
// of them, one per CU. Together and apart, top-k 20: 2 rows 9.2 and 10.8 us, 16
// rows 10.1 and 11.6, 24 rows 17.2 and 12.5.
constexpr int FIND_ROWS = 16;
constexpr float LEAST_TEMPERATURE = 0x1p-100f;
constexpr float FLT_MAX = 3.402823466e38f;

// An integer that orders floats (a NaN as minus infinity).
__device__ __forceinline__ unsigned order_key(float x)
{
    if (x != x) x = -INFINITY;
    if (x == 0.f) x = 0.f; // the two zeros are equal
    const unsigned b = __builtin_bit_cast(unsigned, x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

struct RowSettings {
    float max, half_max, per_bin; // (128 / T, see bin_of)
    float floor;        // no value below it, and no NaN, has a bin
    double weigh_max, weigh, scale, min_p; // weigh: 1024 / (T ln 2)
};
// The bin of a value from the row's floor on, SAMPLE_BINS where its weight is zero.
// (Rounding is monotone, so larger values never have larger bins. Half the
// difference, which no two values' overflows. Where the maximum is infinite its
// difference with itself is a NaN, whose maximum with zero is zero, and every
// other value's is infinite.)
__device__ __forceinline__ int bin_of(float l, const RowSettings &s)
{
    return (int)fminf(fmaxf(fmaf(-0.5f, l, s.half_max) * s.per_bin, 0.f), (float)SAMPLE_BINS);
}
// A value below which bins are larger than `hi`: the border of hi + 1, less
// what the rounding of bin_of's difference and product can move it by.
__device__ __forceinline__ float bin_floor(int hi, const RowSettings &s)
{
    if (s.max == INFINITY) return s.max;
    const float d = (float)(hi + 1) / s.per_bin; // (half, as in bin_of)
    const float f = s.half_max - d - (fabsf(s.half_max) + d) * 1e-6f;
    return fmaxf(2.f * f, -FLT_MAX); // (minus infinity has no bin)
}

// The bin of any value.
__device__ __forceinline__ int bin_at(float l, const RowSettings &s)
{
    return l >= s.floor ? bin_of(l, s) : SAMPLE_BINS;
}
// 2^(i / 64), rounded to 64 bits.
__constant__ const double EXP2_64[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};
// 2^(i / 1024).
__constant__ const double EXP2_1024[16] = {
    1.0, 1.0006771306930664, 1.0013547198921082, 1.002032767907594,
    1.0027112750502025, 1.0033902416308227, 1.004069667960554, 1.0047495543507072,
    1.0054299011128027, 1.006110708558573, 1.0067919769999607, 1.0074737067491204,
    1.0081558981184175, 1.0088385514204294, 1.0095216669679448, 1.0102052450739643};
// The table 2^(i / 1024) in LDS (ends with a barrier).
constexpr int SAMPLE_TABLE = 1024;
__device__ __forceinline__ void load_table(double *table)
{
    static_assert(SAMPLE_TABLE == SAMPLE_THREADS, "an entry per thread");
    table[threadIdx.x] = EXP2_64[threadIdx.x >> 4] * EXP2_1024[threadIdx.x & 15];
    __syncthreads();
}
// The weight of a value that has a bin: exp((l - max) / T) = 2^(y / 1024) with
// y = (l - max) 1024 / (T ln 2) in [-48800, 0], y = n + f with n whole and
// |f| <= 1/2: 2^(n >> 10), by the exponent, times the table's 2^((n & 1023) /
// 1024) times 2^(f / 1024), whose series to f^3 is off by less than 6e-16 (the
// first term left out, (ln 2 / 2048)^4 / 24) where a unit of the sums is 2^-46 =
// 1.4e-14. n comes of adding 1.5 2^52, whose low bits then hold it. Ten 64-bit
// operations a value, and those are what bounds a pass that weighs every value:
// 18 of them (a table of 64, a series to r^5, n by rounding and conversion)
// made the sums' pass over 64 rows of 128167 17.2 us instead of 16.4.
__device__ __forceinline__ double weight(float l, const RowSettings &s, const double *table)
{
    constexpr double WHOLE = 6755399441055744.0, LN2 = 0.6931471805599453 / SAMPLE_TABLE;
    const double d = (double)fminf(l, FLT_MAX) - s.weigh_max; // (inf and inf: 0)
    const double t = fma(d, s.weigh, WHOLE), f = fma(d, s.weigh, WHOLE - t);
    const int n = (int)(unsigned)__builtin_bit_cast(u64, t);
    double e = fma(f, LN2 * LN2 * LN2 / 6, LN2 * LN2 / 2);
    e = fma(e, f, LN2);
    e = fma(e, f, 1.0) * table[n & (SAMPLE_TABLE - 1)];
    const u64 bits = __builtin_bit_cast(u64, e) + ((u64)(unsigned)(n >> 10) << 52);
    return __builtin_bit_cast(double, bits); // (e >= 0.99, n >> 10 >= -48: no underflow)
}
// w 2^shift as an integer, to nearest: the sum with 2^52 holds it in its low
// bits (w 2^shift <= 2^46).
__device__ __forceinline__ u64 fixed(double w, const RowSettings &s)
{
    return __builtin_bit_cast(u64, fma(w, s.scale, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
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
    int vocab, shift, splits, run; // run: values of each of a split's 16 runs
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *random;
    int *token;
    float *prob;
    // scratch
    float *smax;     // [rows][splits]
    unsigned *count; // [rows][splits][SAMPLE_BINS]
    u64 *wsum;       // [rows][splits][SAMPLE_BINS]
    u64 *sums;       // [rows][splits][16]: a run's weight in the bins before the listed ones
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
    int split;          // the first split that holds the maximum
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
    r.max = wave::max64(m);
    r.split = __ffsll((long long)__ballot(m == r.max)) - 1;
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
    r.st.half_max = 0.5f * r.max;
    // (so that bins of 1/64 are numbers; equal maxima share what there is)
    const double inv_t = 1.0 / (double)fmaxf(temp, LEAST_TEMPERATURE);
    r.st.per_bin = (float)(128.0 * inv_t);
    r.st.weigh_max = fminf(r.max, FLT_MAX);
    r.st.weigh = inv_t * (SAMPLE_TABLE * 1.4426950408889634);
    r.st.scale = ldexp(1.0, a.shift);
    r.st.floor = bin_floor(SAMPLE_BINS - 1, r.st);
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

// f(value, index, whether it counts) for a thread's values of [begin, end): eight
// loads in flight, then four calls at a time from one place in the code. (A
// launch starts with a cold instruction cache: f's 64-bit exponential is not
// fetched eight times over.) Values below `floor`, and NaNs, do not count: where
// a wave's are all so, as most are when few can be kept, a step is its loads
// and a comparison each.
template <class F>
__device__ __forceinline__ void each_value(const float *x, int begin, int end, int first, int step,
                                           float floor, F f)
{
    for (int i = begin + first; i < end; i += 8 * step) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = x[min(i + u * step, end - 1)];
        bool any = false;
#pragma unroll
        for (int u = 0; u < 8; ++u) any |= v[u] >= floor;
        if (!__any(any)) continue;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = i + (4 * h + u) * step;
                f(v[u], j, j < end && v[u] >= floor);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = v[u + 4];
        }
    }
}

// ---- max ----
// (v_max ignores a NaN)
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_max_kernel(SampleArgs a)
{
    __shared__ float sm[SAMPLE_WAVES];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const float *x = a.logits + (size_t)row * a.vocab;
    const int per = SAMPLE_WAVES * a.run, end = min(a.vocab, (s + 1) * per);
    float mx = -INFINITY;
    for (int i = s * per + t; i < end; i += 8 * SAMPLE_THREADS) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = x[min(i + u * SAMPLE_THREADS, end - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u) mx = fmaxf(mx, v[u]);
    }
    mx = wave::max64(mx);
    if ((t & 63) == 0) sm[t >> 6] = mx;
    __syncthreads();
    if (t < 64) {
        mx = wave::max64(sm[t & (SAMPLE_WAVES - 1)]);
        if (t == 0) {
            a.smax[row * a.splits + s] = mx;
            if (s == 0) a.have[2 * row] = a.have[2 * row + 1] = 0;
        }
    }
}

// ---- bins ----
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_bins_kernel(SampleArgs a)
{
    __shared__ u64 hw[SAMPLE_BINS];
    __shared__ unsigned hc[SAMPLE_BINS];
    __shared__ double table[SAMPLE_TABLE];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x;
    const RowPlan r = plan_row(a, row);
    if (!r.counts && !r.sums) return;
    if (r.sums) load_table(table);
    const float *x = a.logits + (size_t)row * a.vocab;
    const int per = SAMPLE_WAVES * a.run, end = min(a.vocab, (s + 1) * per);
    for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
        hw[b] = 0;
        hc[b] = 0;
    }
    __syncthreads();
    each_value(x, s * per, end, t, SAMPLE_THREADS, r.st.floor, [&](float v, int, bool counts) {
        const int b = bin_of(v, r.st);
        if (!counts || b >= SAMPLE_BINS) return;
        if (r.counts) atomicAdd(hc + b, 1u);
        if (r.sums) atomicAdd(hw + b, fixed(weight(v, r.st, table), r.st));
    });
    __syncthreads();
    const size_t at = ((size_t)row * a.splits + s) * SAMPLE_BINS;
    for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
        if (r.counts) a.count[at + b] = hc[b];
        if (r.sums) a.wsum[at + b] = hw[b];
    }
}

// ---- find ----
// f, in LDS: what the row's histogram says, by a workgroup. (Ends with a barrier.)
__device__ __forceinline__ void find_cuts(const SampleArgs &a, const RowPlan &r, int row, Found &f,
                                          u64 *wsum)
{
    const int t = threadIdx.x;
    // (nothing cut: all bins summed)
    if (t == 0) f = Found{SAMPLE_BINS, SAMPLE_BINS, -1, 0, 0, 0, 0, 0, 0};
    if (r.counts || r.sums) {
        // this thread's two bins over all splits, and their running totals
        u64 c0 = 0, c1 = 0, w0 = 0, w1 = 0, ctotal = 0, wtotal = 0;
        const size_t at = (size_t)row * a.splits * SAMPLE_BINS + 2 * t;
        if (r.counts) {
#pragma unroll 8
            for (int i = 0; i < a.splits; ++i) {
                const uint2 c =
                    *reinterpret_cast<const uint2 *>(a.count + at + (size_t)i * SAMPLE_BINS);
                c0 += c.x;
                c1 += c.y;
            }
        }
        if (r.sums) {
#pragma unroll 8
            for (int i = 0; i < a.splits; ++i) {
                const ulonglong2 w =
                    *reinterpret_cast<const ulonglong2 *>(a.wsum + at + (size_t)i * SAMPLE_BINS);
                w0 += w.x;
                w1 += w.y;
            }
        }
        const u64 cup = block_scan(c0 + c1, wsum, &ctotal);
        const u64 wup = r.sums ? block_scan(w0 + w1, wsum, &wtotal) : 0;
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
}
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_find_kernel(SampleArgs a)
{
    __shared__ u64 wsum[SAMPLE_WAVES];
    __shared__ Found f;
    const int row = blockIdx.x;
    const RowPlan r = plan_row(a, row);
    if (r.greedy) return;
    find_cuts(a, r, row, f, wsum);
    if (threadIdx.x == 0) a.found[row] = f;
}

// ---- sums ----
// FIND: every split finds the cuts for itself, without the launch before (see
// FIND_ROWS).
template <bool FIND>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_sums_kernel(SampleArgs a)
{
    __shared__ unsigned listed[2], base[2];
    __shared__ u64 list[2][SAMPLE_LIST];
    __shared__ double table[SAMPLE_TABLE];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const RowPlan r = plan_row(a, row);
    if (r.greedy) return;
    Found g;
    if (FIND) {
        __shared__ u64 wsum[SAMPLE_WAVES];
        __shared__ Found f;
        find_cuts(a, r, row, f, wsum);
        g = f;
        if (s == 0 && t == 0) a.found[row] = f;
    } else {
        g = a.found[row];
    }
    if (t < 2) listed[t] = 0;
    load_table(table);
    const float *x = a.logits + (size_t)row * a.vocab;
    const int begin = min(a.vocab, (s * SAMPLE_WAVES + wave) * a.run);
    const int end = min(a.vocab, begin + a.run);
    u64 sum = 0;
    const float least = bin_floor(min(max(g.hi, g.kbin), SAMPLE_BINS - 1), r.st);
    each_value(x, begin, end, lane, 64, least, [&](float v, int j, bool counts) {
        const int b = bin_of(v, r.st);
        counts = counts && b < SAMPLE_BINS;
        if (g.lo > 0) { // (no branch by value: a wave's values are mixed)
            const double w = weight(v, r.st, table);
            const u64 x = fixed(w, r.st);
            sum += counts && b < g.lo && w >= r.st.min_p ? x : 0;
        }
        const bool in0 = counts && b >= g.lo && b <= g.hi, in1 = counts && b == g.kbin;
        if (in0 || in1) {
            const int which = in0 ? 0 : 1;
            const unsigned n = atomicAdd(listed + which, 1u);
            if (n < SAMPLE_LIST) list[which][n] = (u64)order_key(v) << 32 | (unsigned)~j;
        }
    });
    sum = wave_sum(sum);
    if (lane == 0) a.sums[((size_t)row * a.splits + s) * SAMPLE_WAVES + wave] = sum;
    __syncthreads();
    if (t < 2) base[t] = listed[t] ? atomicAdd(a.have + 2 * row + t, listed[t]) : 0;
    __syncthreads();
#pragma unroll 1
    for (int which = 0; which < 2; ++which)
        for (unsigned n = t; n < min(listed[which], (unsigned)SAMPLE_LIST); n += SAMPLE_THREADS)
            if (base[which] + n < SAMPLE_LIST)
                a.list[((size_t)row * 2 + which) * SAMPLE_LIST + base[which] + n] = list[which][n];
}

// ---- draw ----
__device__ __forceinline__ float value_of(u64 key) // the float of an order key
{
    const unsigned k = (unsigned)(key >> 32);
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The whole row by one workgroup (see the head of the file).
__device__ __forceinline__ void row_alone(const SampleArgs &a, const RowPlan &plan, int row,
                                          const double *table, u64 *hw, unsigned *hc, u64 *wsum,
                                          u64 *pick)
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
        const int b = bin_at(v, st);
        if (b < SAMPLE_BINS) {
            atomicAdd(hc + b, 1u);
            atomicAdd(hw + b, fixed(weight(v, st, table), st));
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
                if (bin_at(v, st) != b) continue;
                atomicAdd(hc + ((key >> sh) & 255), 1u);
                atomicAdd(hw + ((key >> sh) & 255), fixed(weight(v, st, table), st));
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
        if (bin_at(v, st) >= SAMPLE_BINS) return 0;
        const double w = weight(v, st, table);
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
                            (float)(weight(x[b + lane], st, table) * st.scale / (double)whole);
                }
                break;
            }
            before = __shfl(upto, 63, 64);
        }
    }
}


// Cuts a list in LDS, whose keys lie in `range`, by a workgroup: finds the
// smallest key of the order's shortest prefix that has `count` members or the
// weight `target` (the other one is unbounded); at most all n members.
// *weight_of: that prefix's weight. Digits of 8 bits, largest first: a histogram
// of the members that share the digits so far, of which one wave finds the digit
// where the prefix ends, until 64 members are left, which are ranked against each
// other (going on to a single one took up to two more digits: a launch of two cuts
// of 1000 members 18.5 -> 17.1 us, and 15.1 with the keys' range found while they
// are loaded).
struct ListScratch {
    u64 hw[256];
    u64 rank[64];           // of the members ranked: the weight before them
    unsigned hc[256], left; // left: their number
    u64 out[4]; // digit, members before it, weight before it, members in it
};
__device__ __forceinline__ u64 cut_list(const u64 *key, const u64 *w, int n, const u64 *range,
                                        u64 count, u64 target, ListScratch &l, u64 *weight_of)
{
    const int t = threadIdx.x, lane = t & 63;
    // keys relative to the smallest, from the highest bit in which they differ
    // (members of few bins share theirs: a first digit of one value would be a
    // histogram of one bin)
    const u64 kmin = range[0], span = range[1] - kmin;
    const int top = max(0, (span ? 63 - __clzll((long long)span) : 0) - 7);
    u64 prefix = 0, before = 0, wbefore = 0;
    int last = top + 8; // the bits from here on are `prefix`
    for (int sh = top;; sh = max(0, sh - 8)) {
        __syncthreads();
        if (t < 256) {
            l.hw[t] = 0;
            l.hc[t] = 0;
        }
        if (t == 0) l.left = 0;
        __syncthreads();
        for (int i = t; i < n; i += SAMPLE_THREADS)
            if (const u64 k = key[i] - kmin; sh == top || k >> last == prefix) {
                const int d = (int)((k >> sh) & ((1u << (last - sh)) - 1));
                atomicAdd(l.hc + d, 1u);
                atomicAdd(l.hw + d, w[i]);
            }
        __syncthreads();
        if (t < 64) { // lane: digits 255 - 4 lane .. 252 - 4 lane
            u64 c[4], v[4], cs = 0, vs = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                cs += c[i] = l.hc[255 - 4 * lane - i];
                vs += v[i] = l.hw[255 - 4 * lane - i];
            }
            u64 cb = before + wave_scan(cs, lane) - cs, vb = wbefore + wave_scan(vs, lane) - vs;
            // the digit that reaches the cut, else the last that has members
            int at = -1;
            u64 ac = 0, av = 0, am = 0;
            bool ends = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!ends && c[i]) {
                    at = 255 - 4 * lane - i;
                    ac = cb;
                    av = vb;
                    am = c[i];
                    ends = cb + c[i] >= count || vb + v[i] >= target;
                }
                cb += c[i];
                vb += v[i];
            }
            const u64 end = __ballot(ends), any = __ballot(at >= 0);
            const int pick = end ? __ffsll((long long)end) - 1 : 63 - __clzll((long long)any);
            if (lane == pick) {
                l.out[0] = at;
                l.out[1] = ac;
                l.out[2] = av;
                l.out[3] = am;
            }
        }
        __syncthreads();
        prefix = prefix << (last - sh) | l.out[0];
        before = l.out[1];
        wbefore = l.out[2];
        last = sh;
        if (l.out[3] <= 64) { // (one at the last digit: keys differ)
            for (int i = t; i < n; i += SAMPLE_THREADS)
                if ((key[i] - kmin) >> sh == prefix) {
                    const unsigned at = atomicAdd(&l.left, 1u);
                    l.hw[2 * at] = key[i];
                    l.hw[2 * at + 1] = w[i];
                }
            if (t < 64) {
                l.hc[t] = (unsigned)before; // (the members before each, and their weight)
                l.rank[t] = wbefore;
            }
            __syncthreads();
            // each wave holds the members, one per lane, against a sixteenth of them
            const int m = l.left;
            const u64 k = lane < m ? l.hw[2 * lane] : 0, x = lane < m ? l.hw[2 * lane + 1] : 0;
            unsigned larger = 0;
            u64 sum = 0;
            for (int j = t >> 6; j < m; j += SAMPLE_WAVES)
                if (l.hw[2 * j] > k) {
                    ++larger;
                    sum += l.hw[2 * j + 1];
                }
            atomicAdd(l.hc + lane, larger);
            atomicAdd(l.rank + lane, sum);
            __syncthreads();
            if (t < 64) {
                const u64 c = l.hc[lane], v = l.rank[lane];
                const bool open = lane < m && c < count && v < target;
                const bool ends = open && (c + 1 >= count || v + x >= target);
                // (reached by none: the last)
                const bool is = __any(ends) ? ends : open && c == before + m - 1;
                if (is) {
                    l.out[0] = k;
                    l.out[1] = v + x;
                }
            }
            __syncthreads();
            prefix = l.out[0];
            *weight_of = l.out[1];
            __syncthreads();
            return prefix;
        }
    }
}

// The value of lane l, uniform.
__device__ __forceinline__ u64 lane64(u64 v, int l)
{
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)v, l);
}

__global__ __launch_bounds__(SAMPLE_THREADS) void sample_draw_kernel(SampleArgs a)
{
    __shared__ u64 key[SAMPLE_LIST], lw[SAMPLE_LIST]; // a list's keys and weights
    __shared__ ListScratch ls;
    __shared__ u64 wsum[SAMPLE_WAVES], pick[4];
    __shared__ u64 range[2][2]; // of list 1's keys, and list 0's
    __shared__ u64 run_sum[SAMPLE_SPLITS * SAMPLE_WAVES];
    __shared__ double table[SAMPLE_TABLE];
    static_assert(SAMPLE_SPLITS * SAMPLE_WAVES <= SAMPLE_THREADS, "a run per thread");
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const Found f = a.found[row];
    const unsigned n0 = a.have[2 * row], n1 = a.have[2 * row + 1];
    const u64 *lists = a.list + (size_t)row * 2 * SAMPLE_LIST;
    const u64 first_key = lists[lane]; // (of list 0: a small list's members)
    const float random = a.random[row];
    const RowPlan r = plan_row(a, row);
    if (r.greedy) { // the first maximum, or nothing to take
        const bool any = r.max > -INFINITY;
        if (t == 0) pick[0] = 0x7fffffff;
        __syncthreads();
        if (any) {
            const int per = SAMPLE_WAVES * a.run, end = min(a.vocab, (r.split + 1) * per);
            int first = 0x7fffffff;
            for (int i = r.split * per + t; i < end; i += 8 * SAMPLE_THREADS) {
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    v[u] = a.logits[(size_t)row * a.vocab + min(i + u * SAMPLE_THREADS, end - 1)];
#pragma unroll
                for (int u = 7; u >= 0; --u) // (past the end: the last value again)
                    if (v[u] == r.max)
                        first = min(first, min(i + u * SAMPLE_THREADS, end - 1));
            }
            if (first != 0x7fffffff) atomicMin(pick, (u64)first);
        }
        __syncthreads();
        if (t == 0) {
            a.token[row] = any ? (int)pick[0] : -1;
            if (a.prob) a.prob[row] = any ? 1.f : 0.f;
        }
        return;
    }
    const RowSettings &st = r.st;
    if (t < 2) {
        range[t][0] = ~(u64)0;
        range[t][1] = 0;
    }
    load_table(table);
    if (n0 > SAMPLE_LIST || n1 > SAMPLE_LIST) {
        static_assert(SAMPLE_LIST >= SAMPLE_BINS, "its histograms' place");
        row_alone(a, r, row, table, key, (unsigned *)lw, wsum, pick);
        return;
    }
    // Every kept value in a list of a wave: a member per lane, the members with
    // larger keys counted and weighed by readlane.
    if (f.lo == 0 && f.kbin < 0 && n0 <= 64) {
        if (wave) return;
        const int n = n0;
        const bool in = lane < n;
        const u64 k = in ? first_key : 0;
        const double wd = in ? weight(value_of(k), st, table) : 0.0;
        u64 w = fixed(wd, st);
        int rank = 0;
        u64 before = 0;
        for (int j = 0; j < n; ++j) {
            const bool larger = lane64(k, j) > k;
            rank += larger;
            before += larger ? lane64(w, j) : 0;
        }
        bool keep = in && (!f.k_in_list || rank < r.k);
        const u64 of = f.k_in_list ? wave_sum(keep ? w : 0) : f.total;
        if (r.by_p) keep = keep && before < top_p_target(r.p, of);
        keep = keep && wd >= st.min_p;
        w = keep ? w : 0;
        const u64 whole = wave_sum(w), target = draw_target(random, whole);
        u64 upto = 0; // the kept weights up to this index
        for (int j = 0; j < n; ++j)
            upto += (unsigned)lane64(k, j) >= (unsigned)k ? lane64(w, j) : 0;
        int token = keep && upto >= target ? (int)~(unsigned)k : 0x7fffffff;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) token = min(token, __shfl_xor(token, o, 64));
        if (in && (int)~(unsigned)k == token) {
            a.token[row] = token;
            if (a.prob) a.prob[row] = (float)(wd * st.scale / (double)whole);
        }
        return;
    }
    // First the weight that top-p is of, where the top-k's cut lies behind the
    // list that top-p cuts; then the top-k's cut in that list, then top-p's.
    // kept: the keys from `last` on. (One place in the code for the three cuts.)
    u64 of = f.total, last = 0;
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {
        const int n = step ? n0 : n1;
        if (step < 2 && (step || f.kbin >= 0)) { // (a list and its weights)
            __syncthreads();
            u64 least = ~(u64)0, most = 0;
            for (int i = t; i < n; i += SAMPLE_THREADS) {
                const u64 k = lists[(step ? 0 : 1) * SAMPLE_LIST + i];
                key[i] = k;
                lw[i] = fixed(weight(value_of(k), st, table), st);
                least = min(least, k);
                most = max(most, k);
            }
            if (wave * 64 < n) {
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    least = min(least, (u64)__shfl_xor(least, o, 64));
                    most = max(most, (u64)__shfl_xor(most, o, 64));
                }
                if (lane == 0) {
                    atomicMin(range[step], least);
                    atomicMax(range[step] + 1, most);
                }
            }
            __syncthreads();
        }
        if (n == 0 || !(step == 0 ? f.kbin >= 0 : step == 1 ? f.k_in_list : r.by_p)) continue;
        constexpr u64 ALL = ~(u64)0;
        u64 in;
        const u64 cut = cut_list(key, lw, n, range[min(step, 1)],
                                 step == 0 ? r.k - f.kbefore : step == 1 ? r.k - f.before : ALL,
                                 step < 2 ? ALL : top_p_target(r.p, max(of, (u64)1)) - f.wbefore, ls,
                                 &in);
        if (step < 2) of = (step ? f.wbefore : f.kwbefore) + in;
        if (step) last = max(last, cut);
    }
    // the kept members' weights to their runs
    const int runs = a.splits * SAMPLE_WAVES;
    if (t < runs) run_sum[t] = a.sums[(size_t)row * runs + t];
    __syncthreads();
    for (int i = t; i < (int)n0; i += SAMPLE_THREADS)
        if (key[i] >= last && weight(value_of(key[i]), st, table) >= st.min_p)
            atomicAdd(run_sum + (int)(~(unsigned)key[i]) / a.run, lw[i]);
    __syncthreads();
    // the run that holds the target, and the token in it
    u64 whole;
    const u64 mine = t < runs ? run_sum[t] : 0, upto = block_scan(mine, wsum, &whole);
    const u64 target = draw_target(random, whole);
    if (upto >= target && upto - mine < target) {
        pick[0] = t;
        pick[1] = upto - mine;
    }
    __syncthreads();
    const float *x = a.logits + (size_t)row * a.vocab;
    const int begin = (int)pick[0] * a.run, end = min(a.vocab, begin + a.run);
    u64 before = pick[1];
#pragma unroll 1
    for (int b = begin; b < end; b += SAMPLE_THREADS) {
        const int i = b + t;
        u64 w = 0, all;
        double wd = 0.0;
        if (i < end) {
            const float v = x[i];
            const int bin = bin_at(v, st);
            if (bin < SAMPLE_BINS && bin <= f.hi &&
                (bin < f.lo || ((u64)order_key(v) << 32 | (unsigned)~i) >= last)) {
                wd = weight(v, st, table);
                if (wd >= st.min_p) w = fixed(wd, st);
            }
        }
        const u64 up = before + block_scan(w, wsum, &all);
        if (up >= target && up - w < target) {
            a.token[row] = i;
            if (a.prob) a.prob[row] = (float)(wd * st.scale / (double)whole);
        }
        before += all;
        if (before >= target) break;
    }
}

struct SampleLayout {
    int splits, run;
    size_t count, wsum, sums, found, have, list, bytes;
};
// Splits: as many workgroups as fill the GPU twice (64 rows: 57.4 us; filled once
// 60.1, four times 61.4), but at most 16 (each workgroup of the third launch adds
// up all of a row's histograms; two rows, as five launches: 21.9 us, with 8 23.1,
// with 32 23.6) and
// none of fewer than 1024 values.
SampleLayout sample_layout(int rows, int vocab)
{
    SampleLayout l;
    const int most = (vocab + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
    l.splits = std::max(1, std::min({512 / rows, SAMPLE_SPLITS, most}));
    const int runs = l.splits * SAMPLE_WAVES;
    l.run = ((vocab + runs - 1) / runs + 63) / 64 * 64;
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t n = (size_t)rows * l.splits;
    l.count = up(n * 4);
    l.wsum = l.count + n * SAMPLE_BINS * 4;
    l.sums = l.wsum + n * SAMPLE_BINS * 8;
    l.found = l.sums + up(n * SAMPLE_WAVES * 8);
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
    a.run = l.run;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.random = random;
    a.token = token;
    a.prob = prob;
    a.smax = (float *)base;
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
    if (rows <= FIND_ROWS) {
        hipLaunchKernelGGL(sample_sums_kernel<true>, grid, block, 0, st, a);
    } else {
        hipLaunchKernelGGL(sample_find_kernel, dim3(rows), block, 0, st, a);
        hipLaunchKernelGGL(sample_sums_kernel<false>, grid, block, 0, st, a);
    }
    hipLaunchKernelGGL(sample_draw_kernel, dim3(rows), block, 0, st, a);
    return (int)hipGetLastError();
}

} // namespace hyq
