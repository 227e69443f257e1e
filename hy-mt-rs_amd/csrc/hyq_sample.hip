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
// as integers w_i 2^SHIFT, so that their sums are exact and do not depend on
// the order of addition: histograms by atomics give the same bits always, and
// a border falls where 64-bit arithmetic puts it. Weights below 2^-SHIFT-1 of
// the largest are zero and never drawn (SHIFT is 62 minus log2 of the
// vocabulary, at most 46).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef unsigned long long u64;

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_WAVES = SAMPLE_THREADS / 64;
constexpr int SAMPLE_BINS = 2048;

// An integer that orders floats (a NaN as minus infinity).
__device__ __forceinline__ unsigned order_key(float x)
{
    if (x != x) x = -INFINITY;
    if (x == 0.f) x = 0.f; // the two zeros are equal
    const unsigned b = __builtin_bit_cast(unsigned, x);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

struct RowSettings {
    float max;
    double inv_t, scale, min_p;
};
__device__ __forceinline__ double weight(float l, const RowSettings &s)
{
    if (l == s.max) return 1.0;
    if (!(l > -INFINITY) || s.max == INFINITY) return 0.0;
    return exp(((double)l - (double)s.max) * s.inv_t);
}
__device__ __forceinline__ u64 fixed(double w, const RowSettings &s)
{
    return (u64)(w * s.scale + 0.5);
}
// Bins of (max - l) / T, 1/64 wide; the last takes all that is further away.
__device__ __forceinline__ int bin_of(float l, const RowSettings &s)
{
    if (l == s.max) return 0;
    const double d = ((double)s.max - (double)l) * s.inv_t * 64.0;
    return d < SAMPLE_BINS - 1 ? (int)d : SAMPLE_BINS - 1;
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

__global__ __launch_bounds__(SAMPLE_THREADS) void sample_row_kernel(
    const float *__restrict__ logits, int vocab, int shift, const float *__restrict__ temperature,
    const int *__restrict__ top_k, const float *__restrict__ top_p,
    const float *__restrict__ min_p, const float *__restrict__ random, int *__restrict__ token,
    float *__restrict__ prob)
{
    __shared__ u64 hw[SAMPLE_BINS];
    __shared__ unsigned hc[SAMPLE_BINS];
    __shared__ u64 wsum[SAMPLE_WAVES];
    __shared__ float smax[SAMPLE_WAVES];
    __shared__ int sidx[SAMPLE_WAVES];
    __shared__ u64 pick[4];
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const float *x = logits + (size_t)row * vocab;

    // the largest value and its first index
    float mx = -INFINITY;
    int mi = 0x7fffffff;
    for (int i = t; i < vocab; i += SAMPLE_THREADS) {
        const float v = x[i];
        if (v > mx) {
            mx = v;
            mi = i;
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
    if (lane == 0) {
        smax[wave] = mx;
        sidx[wave] = mi;
    }
    __syncthreads();
    mx = smax[0];
    mi = sidx[0];
    for (int w = 1; w < SAMPLE_WAVES; ++w)
        if (smax[w] > mx || (smax[w] == mx && sidx[w] < mi)) {
            mx = smax[w];
            mi = sidx[w];
        }
    const float temp = temperature[row];
    if (!(mx > -INFINITY) || !(temp > 0.f)) { // nothing to take, or the first maximum
        if (t == 0) {
            token[row] = mx > -INFINITY ? mi : -1;
            if (prob) prob[row] = mx > -INFINITY ? 1.f : 0.f;
        }
        return;
    }
    RowSettings st;
    st.max = mx;
    st.inv_t = 1.0 / (double)temp;
    st.scale = ldexp(1.0, shift);
    st.min_p = min_p[row] > 0.f ? fmin((double)min_p[row], 1.0) : 0.0;
    const int k = top_k[row];
    const double p = top_p[row];

    for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
        hw[b] = 0;
        hc[b] = 0;
    }
    __syncthreads();
    for (int i = t; i < vocab; i += SAMPLE_THREADS) {
        const float v = x[i];
        const u64 w = fixed(weight(v, st), st);
        if (w) {
            const int b = bin_of(v, st);
            atomicAdd(hc + b, 1u);
            atomicAdd(hw + b, w);
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
                const u64 w = fixed(weight(v, st), st);
                if (!w || bin_of(v, st) != b) continue;
                atomicAdd(hc + ((key >> sh) & 255), 1u);
                atomicAdd(hw + ((key >> sh) & 255), w);
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
        const u64 ties = byw ? (target - before + each - 1) / each : target - before;
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
        const double want = fmax(p, 0.0) * (double)total;
        u64 target = (u64)want;
        if ((double)target < want) ++target;
        target = min(max(target, (u64)1), total);
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
            const double u = fmin(fmax((double)random[row], 0.0), 1.0);
            const double want = u * (double)whole;
            target = min((u64)want + 1, whole); // the first sum > u W is the first >= this
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
                    token[row] = b + lane;
                    if (prob) prob[row] = (float)(weight(x[b + lane], st) * st.scale / (double)whole);
                }
                break;
            }
            before = __shfl(upto, 63, 64);
        }
    }
}

} // namespace

size_t sample_scratch(int rows, int vocab) { return 0; }

int launch_sample(const float *logits, int rows, int vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *random,
                  void *scratch, int *token, float *prob, void *stream)
{
    if (rows <= 0) return 0;
    int bits = 0;
    while ((1ll << bits) < vocab) ++bits;
    const int shift = std::min(46, 62 - bits);
    hipLaunchKernelGGL(sample_row_kernel, dim3(rows), dim3(SAMPLE_THREADS), 0, (hipStream_t)stream,
                       logits, vocab, shift, temperature, top_k, top_p, min_p, random, token, prob);
    return (int)hipGetLastError();
}

} // namespace hyq
