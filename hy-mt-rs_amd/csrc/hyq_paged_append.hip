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

} // namespace

int launch_paged_append(const PagedKv &kv, const float *q, const float *k, const float *v,
                        const float *qn, const float *kn, const float *freq, float eps,
                        bool norm_first, float *q_out, void *stream)
{
    if (kv.rows <= 0) return 0;
    const int groups = (kv.heads + 2 * kv.kvh + 3) / 4;
    const dim3 grid(kv.rows, (groups + 3) / 4);
    hipStream_t st = (hipStream_t)stream;
    if (kv.f16)
        hipLaunchKernelGGL(paged_append_kernel<_Float16>, grid, dim3(256), 0, st, kv, q, k, v, qn,
                           kn, freq, eps, (int)norm_first, q_out);
    else
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, st, kv, q, k, v, qn,
                           kn, freq, eps, (int)norm_first, q_out);
    return (int)hipGetLastError();
}

} // namespace hyq
