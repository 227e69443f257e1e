// New rows of many sequences into a paged KV cache, in one pass: rotation
// (NeoX halves) and per-head RMS norm of q and k in the dense or the hy_v3
// order, q to q_out, k and v to their slots' pages.
//
//   angle_j = p * freq_j, the exact product: it is formed and reduced to
//   [-pi, pi] in 64 bits, so that a far position costs no accuracy (in 32
//   bits the product alone is off by p * 2^-24 radians), and only the
//   reduced angle is rounded to 32 bits.
//   y = x * (w * 1 / sqrt(mean x^2 + eps))
//
// A 16-lane row of a wave takes a head: lane j its dims 4j..4j+3 and
// 64+4j..64+4j+3 as two float4, so the norm's sum is four DPP steps and a wave
// forms four heads at once from one set of angles.
//
// Bound by memory: 2367 rows of 32 + 2 * 8 heads into f32 pages move 116 MB in
// 22.7 us (5.1 TB/s, what a copy reaches), 48 rows of 16 + 2 * 4 heads into f16
// pages take 4.2 to 5 us, a launch and four dependent loads (starts, length,
// page, row).
//
// An 8-bit pool takes, for the 128 numbers x of a head,
//
//   s = max |x| / 127 (rounded to 32 bits), codes c = rint(x / s), x ~ s c,
//
// off by at most s / 2, and by 127 2^-150 more where max |x| < 127 2^-126, whose scale
// is no normal number: its codes are cut to 127, and at 127 2^-150 it is zero. (Of
// numbers at the end of f32's range s is the f32 below, if 127 of it would be
// infinite.) One number that is not finite makes s a NaN, and with it the whole
// head. Keys are formed and divided in 64 bits: a code is the same on
// every run and in every order of summation but where x / s lies within 2^-40 of
// a half, which f32 would make one in 2^15. 2367 rows of 32 + 2 * 8 heads move 89 MB
// in 26 us, bound by the norms, rotations and divisions in 64 bits; 48 rows of 16 + 2 *
// 4 heads take 4.2. Reading the same rows back takes 6.5 us (25 MB), and 2.7.
#include <hip/hip_runtime.h>

#include "hyq_paged.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The slot of packed row `row`: the last one whose first row is <= row among
// those that hold it (a slot without rows holds none); -1 past the last row.
// A count of the starts <= row, 64 of them per load.
__device__ __forceinline__ int slot_of_row(const int *__restrict__ start, int seqs, int row,
                                           int lane)
{
    int n = 0;
    for (int b = 0; b <= seqs; b += 64) {
        const int i = b + lane;
        const bool le = i <= seqs && start[min(i, seqs)] <= row;
        n += __popcll(__ballot(le));
    }
    return n - 1 < seqs ? n - 1 : -1;
}

__device__ __forceinline__ void store4(float *p, const float (&v)[4])
{
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
// (a cached value is rounded to f16 once, here: to nearest, ties to even)
__device__ __forceinline__ void store4(_Float16 *p, const float (&v)[4])
{
    *reinterpret_cast<half4 *>(p) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2],
                                          (_Float16)v[3]};
}

// sin and cos of p * freq (see above); 2 pi is the sum of two doubles, each
// taken off by one fma, so only the fmas' own roundings remain.
__device__ __forceinline__ void angle(int p, float freq, float &sn, float &cs)
{
    const double a = (double)p * (double)freq;
    const double turns = rint(a * 0.15915494309189535);
    const double r = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a));
    sincosf((float)r, &sn, &cs);
}

constexpr double factorial(int n)
{
    double f = 1.;
    for (int i = 2; i <= n; ++i) f *= i;
    return f;
}

// The same in 64 bits: the reduced angle less a multiple of pi / 2 lies within
// pi / 4, where the series of sine and cosine to t^17 and t^18 leave 2^-60.
__device__ __forceinline__ void angle64(int p, float freq, double &sn, double &cs)
{
    const double a = (double)p * (double)freq;
    const double turns = rint(a * 0.15915494309189535);
    const double r = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a));
    const double quarter = rint(r * 0.6366197723675814);
    const double t =
        fma(quarter, -6.123233995736766e-17, fma(quarter, -1.5707963267948966, r));
    const double u = t * t;
    double s = 0., c = 0.; // sums of (-u)^k / (2 k + 1)! and (-u)^k / (2 k)!
#pragma unroll
    for (int k = 9; k >= 0; --k) {
        if (k < 9) s = fma(s, u, (k & 1 ? -1. : 1.) / factorial(2 * k + 1));
        c = fma(c, u, (k & 1 ? -1. : 1.) / factorial(2 * k));
    }
    s *= t;
    const int n = (int)quarter & 3;
    const double x = n & 1 ? c : s, y = n & 1 ? s : c;
    sn = n & 2 ? -x : x;
    cs = (n + 1) & 2 ? -y : y;
}

// Grid (rows, ceil(groups / 4)), four waves: a wave takes a group of four heads,
// in the order query heads, key heads, value heads. (q_out may be q: a thread
// reads what it writes first.)
template <class T>
__global__ __launch_bounds__(256) void paged_append_kernel(
    PagedKv kv, const float *q, const float *__restrict__ k,
    const float *__restrict__ v, const float *__restrict__ qn, const float *__restrict__ kn,
    const float *__restrict__ freq, float eps, int norm_first, float *q_out)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, j = lane & 15;
    const int total = kv.heads + 2 * kv.kvh;
    const int first = (blockIdx.y * 4 + wave) * 4;
    if (first >= total) return;
    const int slot = slot_of_row(kv.start, kv.seqs, row, lane);
    if (slot < 0) return; // a row behind the last slot's
    const int begin = kv.start[slot], end = min(kv.start[slot + 1], kv.rows);
    const int pos = kv.len[slot] - (end - begin) + (row - begin);
    // where the row's key and value go: nowhere when the table names no page
    T *dst = nullptr;
    if (pos >= 0 && (pos >> kv.shift) < kv.stride) {
        const int page = kv.table[(size_t)slot * kv.stride + (pos >> kv.shift)];
        const size_t head = (size_t)KV_D << kv.shift;
        if (page >= 0 && page < kv.npages)
            dst = (T *)const_cast<void *>(kv.pages) + (size_t)page * 2 * kv.kvh * head +
                  (size_t)(pos & ((1 << kv.shift) - 1)) * KV_D;
    }
    float sn[4], cs[4];
    if (first < kv.heads + kv.kvh) {
        const float4 f = *reinterpret_cast<const float4 *>(freq + 4 * j);
        angle(pos, f.x, sn[0], cs[0]);
        angle(pos, f.y, sn[1], cs[1]);
        angle(pos, f.z, sn[2], cs[2]);
        angle(pos, f.w, sn[3], cs[3]);
    }
    const int h = first + (lane >> 4);
    if (h < total) {
        const bool is_q = h < kv.heads, is_v = h >= kv.heads + kv.kvh;
        const int kh = h - kv.heads - (is_v ? kv.kvh : 0);
        const float *src = is_q ? q + ((size_t)row * kv.heads + h) * KV_D
                                : (is_v ? v : k) + ((size_t)row * kv.kvh + kh) * KV_D;
        // (read once: prompts of 2367 rows 24.2 -> 22.9 us)
        const f32x4 a4 = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(src + 4 * j));
        const f32x4 b4 =
            __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(src + 64 + 4 * j));
        float a[4] = {a4[0], a4[1], a4[2], a4[3]}, b[4] = {b4[0], b4[1], b4[2], b4[3]};
        if (!is_v) {
            const float *w = is_q ? qn : kn;
            const float4 wa = *reinterpret_cast<const float4 *>(w + 4 * j);
            const float4 wb = *reinterpret_cast<const float4 *>(w + 64 + 4 * j);
            const float w0[4] = {wa.x, wa.y, wa.z, wa.w}, w1[4] = {wb.x, wb.y, wb.z, wb.w};
            auto turn = [&]() {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = a[i] * cs[i] - b[i] * sn[i];
                    b[i] = a[i] * sn[i] + b[i] * cs[i];
                    a[i] = x;
                }
            };
            auto norm = [&]() {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
                const float scale = 1.0f / sqrtf(wave::sum16(ss) / (float)KV_D + eps);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] *= w0[i] * scale;
                    b[i] *= w1[i] * scale;
                }
            };
            if (norm_first) {
                norm();
                turn();
            } else {
                turn();
                norm();
            }
        }
        if (is_q) {
            float *o = q_out + ((size_t)row * kv.heads + h) * KV_D + 4 * j;
            store4(o, a);
            store4(o + 64, b);
        } else if (dst) {
            T *o = dst + ((size_t)((is_v ? kv.kvh : 0) + kh) * KV_D << kv.shift) + 4 * j;
            store4(o, a);
            store4(o + 64, b);
        }
    }
}

// Where packed row `row` lies in the pages: its slot's page, -1 where none, and
// its place in it.
struct Place {
    int slot, pos, page, at;
};
__device__ __forceinline__ Place place_of(const PagedKv &kv, int row, int lane)
{
    Place p;
    p.page = -1;
    p.pos = p.at = 0;
    p.slot = slot_of_row(kv.start, kv.seqs, row, lane);
    if (p.slot < 0) return p; // a row behind the last slot's
    const int begin = kv.start[p.slot], end = min(kv.start[p.slot + 1], kv.rows);
    p.pos = kv.len[p.slot] - (end - begin) + (row - begin);
    p.at = p.pos & ((1 << kv.shift) - 1);
    if (p.pos >= 0 && (p.pos >> kv.shift) < kv.stride) {
        const int page = kv.table[(size_t)p.slot * kv.stride + (p.pos >> kv.shift)];
        if (page >= 0 && page < kv.npages) p.page = page;
    }
    return p;
}

__device__ __forceinline__ double lanes16(double v, int o) { return __shfl_xor(v, o, 16); }

// The codes and the scale of a head's 128 numbers (lane j: 4j .. and 64 + 4j ..)
// to an 8-bit page. row: the position's codes, bias: what is added to them.
__device__ __forceinline__ void store_codes(unsigned char *row, float *scale, const double (&a)[4],
                                            const double (&b)[4], int bias, int j)
{
    double top = 0.;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top = fmax(top, fmax(fabs(a[i]), fabs(b[i])));
        fine = fine && fabs(a[i]) <= 1.7976931348623157e308 && fabs(b[i]) <= 1.7976931348623157e308;
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        top = fmax(top, lanes16(top, o));
        fine = __shfl_xor((int)fine, o, 16) && fine;
    }
    float s = (float)(top / 127.);
    if (top <= 3.4028234663852886e38 && 127.f * s == INFINITY)
        s = __builtin_bit_cast(float, __builtin_bit_cast(int, s) - 1);
    const double inv = s > 0.f ? 1. / (double)s : 0.;
    if (!fine || !(s < INFINITY)) s = __builtin_nanf("");
    auto word = [&](const double (&x)[4]) {
        unsigned w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (a scale of few bits, below 2^-126, may lie under the largest's share)
            const int c = (int)fmin(fmax(rint(x[i] * inv), -127.), 127.); // (a NaN: -127)
            w |= (unsigned)((c + bias) & 255) << (8 * i);
        }
        return w;
    };
    *reinterpret_cast<unsigned *>(row + 4 * j) = word(a);
    *reinterpret_cast<unsigned *>(row + 64 + 4 * j) = word(b);
    if (j == 0) *scale = s;
}

// The append to 8-bit pages: grid and groups as above. A wave's angles are formed
// in 64 bits where it has a key head.
__global__ __launch_bounds__(256) void paged_append_q8_kernel(
    PagedKv kv, const float *q, const float *__restrict__ k, const float *__restrict__ v,
    const float *__restrict__ qn, const float *__restrict__ kn, const float *__restrict__ freq,
    float eps, int norm_first, float *q_out)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, j = lane & 15;
    const int total = kv.heads + 2 * kv.kvh;
    const int first = (blockIdx.y * 4 + wave) * 4;
    if (first >= total) return;
    const Place at = place_of(kv, row, lane);
    if (at.slot < 0) return;
    const int h = first + (lane >> 4);
    if (h >= total) return; // (whole 16-lane rows)
    const bool is_q = h < kv.heads, is_v = h >= kv.heads + kv.kvh;
    const int kh = h - kv.heads - (is_v ? kv.kvh : 0);
    const float *src = is_q ? q + ((size_t)row * kv.heads + h) * KV_D
                            : (is_v ? v : k) + ((size_t)row * kv.kvh + kh) * KV_D;
    const f32x4 a4 = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(src + 4 * j));
    const f32x4 b4 = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(src + 64 + 4 * j));
    // one formation for both widths: `T` numbers, `sum` over the head
    auto formed = [&](auto zero, const float *w, auto angles, auto sum, auto (&a)[4], auto (&b)[4]) {
        typedef decltype(zero) T;
        const float4 f = *reinterpret_cast<const float4 *>(freq + 4 * j);
        const float4 wa = *reinterpret_cast<const float4 *>(w + 4 * j);
        const float4 wb = *reinterpret_cast<const float4 *>(w + 64 + 4 * j);
        const float w0[4] = {wa.x, wa.y, wa.z, wa.w}, w1[4] = {wb.x, wb.y, wb.z, wb.w};
        const float fr[4] = {f.x, f.y, f.z, f.w};
        auto turn = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                T sn, cs;
                angles(at.pos, fr[i], sn, cs);
                const T x = a[i] * cs - b[i] * sn;
                b[i] = a[i] * sn + b[i] * cs;
                a[i] = x;
            }
        };
        auto norm = [&]() {
            T ss = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
            const T scale = T(1) / sqrt(sum(ss) / T(KV_D) + T(eps));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] *= T(w0[i]) * scale;
                b[i] *= T(w1[i]) * scale;
            }
        };
        if (norm_first) {
            norm();
            turn();
        } else {
            turn();
            norm();
        }
    };
    if (is_q) {
        float a[4] = {a4[0], a4[1], a4[2], a4[3]}, b[4] = {b4[0], b4[1], b4[2], b4[3]};
        formed(0.f, qn, angle, [](float x) { return wave::sum16(x); }, a, b);
        float *o = q_out + ((size_t)row * kv.heads + h) * KV_D + 4 * j;
        store4(o, a);
        store4(o + 64, b);
        return;
    }
    if (at.page < 0) return;
    double a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = a4[i];
        b[i] = b4[i];
    }
    if (!is_v)
        formed(0., kn, angle64,
               [](double x) {
#pragma unroll
                   for (int o = 1; o < 16; o <<= 1) x += lanes16(x, o);
                   return x;
               },
               a, b);
    const size_t head = (size_t)KV_D << kv.shift;
    unsigned char *page = (unsigned char *)const_cast<void *>(kv.pages) +
                          (size_t)at.page * 2 * kv.kvh * (head / KV_D * (KV_D + 4));
    const int of = (is_v ? kv.kvh : 0) + kh;
    store_codes(page + of * head + (size_t)at.at * KV_D,
                (float *)(page + 2 * kv.kvh * head) + ((size_t)of << kv.shift) + at.at, a, b,
                is_v ? 128 : 0, j);
}

// The packed rows' keys and values as f32 rows; zeros where no page holds a
// position. Grid (rows, ceil(2 kv_heads / 16)), a 16-lane row a head as above.
// Bound by memory, and for few rows by three dependent loads.
template <class T>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedKv kv, float *__restrict__ k,
                                                         float *__restrict__ v)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, j = lane & 15;
    const int h = (blockIdx.y * 4 + wave) * 4 + (lane >> 4);
    const Place at = place_of(kv, row, lane);
    if (at.slot < 0 || h >= 2 * kv.kvh) return;
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    if (at.page >= 0) {
        const size_t head = (size_t)KV_D << kv.shift;
        if constexpr (sizeof(T) == 1) {
            const unsigned char *page = (const unsigned char *)kv.pages +
                                        (size_t)at.page * 2 * kv.kvh * (head / KV_D * (KV_D + 4));
            const unsigned char *src = page + h * head + (size_t)at.at * KV_D + 4 * j;
            const unsigned wa = *reinterpret_cast<const unsigned *>(src),
                           wb = *reinterpret_cast<const unsigned *>(src + 64);
            const float s =
                ((const float *)(page + 2 * kv.kvh * head))[((size_t)h << kv.shift) + at.at];
            const bool is_v = h >= kv.kvh;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int x = wa >> (8 * i) & 255, y = wb >> (8 * i) & 255;
                a[i] = s * (float)(is_v ? x - 128 : (int)(signed char)x);
                b[i] = s * (float)(is_v ? y - 128 : (int)(signed char)y);
            }
        } else {
            const T *src = (const T *)kv.pages + ((size_t)at.page * 2 * kv.kvh + h) * head +
                           (size_t)at.at * KV_D + 4 * j;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = (float)src[i];
                b[i] = (float)src[64 + i];
            }
        }
    }
    float *o = h < kv.kvh ? k + ((size_t)row * kv.kvh + h) * KV_D
                          : v + ((size_t)row * kv.kvh + h - kv.kvh) * KV_D;
    store4(o + 4 * j, a);
    store4(o + 64 + 4 * j, b);
}

} // namespace

int launch_paged_append(const PagedKv &kv, const float *q, const float *k, const float *v,
                        const float *qn, const float *kn, const float *freq, float eps,
                        bool norm_first, float *q_out, void *stream)
{
    if (kv.rows <= 0) return 0;
    const int groups = (kv.heads + 2 * kv.kvh + 3) / 4;
    const dim3 grid(kv.rows, (groups + 3) / 4);
    hipStream_t st = (hipStream_t)stream;
    if (kv.type == KV_T_Q8)
        hipLaunchKernelGGL(paged_append_q8_kernel, grid, dim3(256), 0, st, kv, q, k, v, qn, kn,
                           freq, eps, (int)norm_first, q_out);
    else if (kv.type == KV_T_F16)
        hipLaunchKernelGGL(paged_append_kernel<_Float16>, grid, dim3(256), 0, st, kv, q, k, v, qn,
                           kn, freq, eps, (int)norm_first, q_out);
    else
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, st, kv, q, k, v, qn,
                           kn, freq, eps, (int)norm_first, q_out);
    return (int)hipGetLastError();
}

int launch_paged_read(const PagedKv &kv, float *k, float *v, void *stream)
{
    if (kv.rows <= 0) return 0;
    const dim3 grid(kv.rows, (2 * kv.kvh + 15) / 16);
    auto kernel = kv.type == KV_T_Q8    ? paged_read_kernel<unsigned char>
                  : kv.type == KV_T_F16 ? paged_read_kernel<_Float16>
                                        : paged_read_kernel<float>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, kv, k, v);
    return (int)hipGetLastError();
}

} // namespace hyq
