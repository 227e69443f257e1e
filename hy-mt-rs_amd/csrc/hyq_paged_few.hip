// Attention over a paged cache for slots of few new rows (decode steps,
// drafted tokens): a stream over the cached keys and values.
//
//   o_r = sum_t 2^(s_rt - m_r) v_t / sum_t 2^(s_rt - m_r),
//   s_rt = log2(e) / sqrt(128) q_r . k_t over the positions t the row sees,
//
// in one pass with the running maximum m_r. The query heads of a KV head and
// its slot's new rows are the up to 16 rows of a matrix tile, so every key and
// value is loaded once for all of them.
//
// A wave works alone: it takes a range of 16-position tiles, holds the rows'
// queries and the 16 x 128 output in registers and loads keys and values
// straight into matrix operands. Products are transposed, so that a lane
// keeps one row (lane % 16) throughout and g = lane / 16 picks positions or
// dims:
//   S^T [16 pos x 16 rows] = K . Q^T, lane: positions 4g .. 4g+3 of its row
//   O^T [dims x 16 rows] += V^T . P^T over four positions per matrix product,
// whose operand P^T [k = g][row] for the positions {4g + e} is exactly what
// the lane holds in element e: no exchange between lanes. Both run on
// v_mfma_f32_16x16x4_f32 (f32 pages: no rounding of anything); f16 pages
// multiply on v_mfma_f32_16x16x32_f16 with q split into f16 high and low
// parts (22 bits of each q, keys exact), and their values are widened.
//
// Work is cut evenly whatever the lengths: the tiles of all (slot, KV head)
// units are numbered in order and worker w of W takes tiles
// [w T / W, (w + 1) T / W). A range that covers a unit whole writes the output,
// a part of one its maximum, sum and unnormalised row to slot w + u (workers
// and units both ascend, so w + u names each pair once), which the merge
// joins in worker order.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged_attn.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int FEW_TILE = 16;
constexpr int FEW_WAVES = 4;

// before[s], in LDS: the tiles of the slots before s over all KV heads, with
// the total at before[seqs]. 256 threads.
struct FewPlan {
    long long total;
    int workers;
};

// (new rows over no positions still have their zeros to be written: one tile)
__device__ __forceinline__ int slot_tiles(const SlotRows &r)
{
    return max(1, (r.len + FEW_TILE - 1) / FEW_TILE);
}
__device__ __forceinline__ int few_tiles(const PagedKv &kv, int s, int few_rows)
{
    const SlotRows r = slot_rows(kv, s);
    return r.n > 0 && r.n <= few_rows ? slot_tiles(r) : 0;
}

__device__ __forceinline__ FewPlan few_plan(const PagedKv &kv, int few_rows, int max_workers,
                                            long long *before, long long *wsum)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    long long carry = 0;
    for (int b = 0; b < kv.seqs; b += 256) {
        const int s = b + t;
        const long long mine = s < kv.seqs ? (long long)few_tiles(kv, s, few_rows) * kv.kvh : 0;
        long long v = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long long u = __shfl_up(v, o, 64);
            if (lane >= o) v += u;
        }
        if (lane == 63) wsum[wave] = v;
        __syncthreads();
        long long base = carry, all = carry;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) base += wsum[w];
            all += wsum[w];
        }
        if (s < kv.seqs) before[s] = base + v - mine;
        carry = all;
        __syncthreads();
    }
    if (t == 0) before[kv.seqs] = carry;
    __syncthreads();
    FewPlan p;
    p.total = carry;
    // two tiles at least for a worker: fewer would only add partial rows
    p.workers = (int)min((long long)max_workers, (carry + 1) / 2);
    return p;
}

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, const f32x4 &c)
{
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f16(const half8 &a, const half8 &b, const f32x4 &c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The operands of one tile, by element type. Dims of an output element
// acc[x][e] (see pv): f32 64 (x / 4) + 16 g + 4 e + x % 4, f16 32 g + 8 e + x.
template <class T> struct Ops;

template <> struct Ops<float> {
    float4 q[8]; // row lane % 16, dims 16 j + 4 g ..
    float4 k[8]; // position lane % 16, the same dims
    float4 v[8]; // position 4 g + x / 2, dims 64 (x % 2) + 4 (lane % 16) ..
    float qscale;
    __device__ __forceinline__ void load_q(const float *row, bool ok, int g)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q[j] = *reinterpret_cast<const float4 *>(row + 16 * j + 4 * g);
            if (!ok) q[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        qscale = 1.f;
    }
    __device__ __forceinline__ void load_k(const float *head, int kpos, int g)
    {
        const float *p = head + (size_t)kpos * KV_D + 4 * g;
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = *reinterpret_cast<const float4 *>(p + 16 * j);
    }
    __device__ __forceinline__ void load_v(const float *head, const int (&vpos)[4], int c)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float *p = head + (size_t)vpos[e] * KV_D + 4 * c;
            v[2 * e] = *reinterpret_cast<const float4 *>(p);
            v[2 * e + 1] = *reinterpret_cast<const float4 *>(p + 64);
        }
    }
    __device__ __forceinline__ f32x4 scores() const
    {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a = mfma_f32(k[j].x, q[j].x, a);
            b = mfma_f32(k[j].y, q[j].y, b);
            a = mfma_f32(k[j].z, q[j].z, a);
            b = mfma_f32(k[j].w, q[j].w, b);
        }
        return a + b;
    }
    __device__ __forceinline__ void pv(const f32x4 &p, f32x4 (&acc)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float4 x = v[2 * e + c];
                acc[4 * c] = mfma_f32(x.x, p[e], acc[4 * c]);
                acc[4 * c + 1] = mfma_f32(x.y, p[e], acc[4 * c + 1]);
                acc[4 * c + 2] = mfma_f32(x.z, p[e], acc[4 * c + 2]);
                acc[4 * c + 3] = mfma_f32(x.w, p[e], acc[4 * c + 3]);
            }
    }
    // 0 where every value of the tile is finite, NaN where one is not
    __device__ __forceinline__ float odd() const
    {
        float z = 0.f;
#pragma unroll
        for (int x = 0; x < 8; ++x)
            z = fmaf(v[x].x, 0.f, fmaf(v[x].y, 0.f, fmaf(v[x].z, 0.f, fmaf(v[x].w, 0.f, z))));
        return z;
    }
    static __device__ __forceinline__ int dim(int x, int e, int g)
    {
        return 64 * (x >> 2) + 16 * g + 4 * e + (x & 3);
    }
    // a lane's four consecutive dims 64 c + 16 g + 4 e ..
    static __device__ __forceinline__ void put(float *o, const f32x4 (&acc)[8], int g, float s)
    {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<float4 *>(o + 64 * c + 16 * g + 4 * e) =
                    make_float4(acc[4 * c][e] * s, acc[4 * c + 1][e] * s, acc[4 * c + 2][e] * s,
                                acc[4 * c + 3][e] * s);
    }
};

template <> struct Ops<_Float16> {
    half8 qh[4], ql[4]; // row lane % 16, dims 32 j + 8 g ..
    half8 k[4];         // position lane % 16, the same dims
    half8 v[4];         // position 4 g + e, dims 8 (lane % 16) ..
    float qscale;
    // q = 2^e (high + low): the row's power of two brings its largest value
    // to [1, 2), inside f16's range whatever the queries' size, and the low
    // part's rounding is 2^-22 of it
    __device__ __forceinline__ void load_q(const float *row, bool ok, int g)
    {
        float x[4][8];
        float mx = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 a = *reinterpret_cast<const float4 *>(row + 32 * j + 8 * g);
            const float4 b = *reinterpret_cast<const float4 *>(row + 32 * j + 8 * g + 4);
            const float t[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[j][i] = ok ? t[i] : 0.f;
                mx = fmaxf(mx, fabsf(x[j][i]));
            }
        }
        mx = wave::max_halves(wave::max_rows2(mx));
        int e = 0;
        if (mx > 0.f && mx < INFINITY) e = ilogbf(mx);
        qscale = ldexpf(1.f, e);
        const float inv = ldexpf(1.f, -e);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[j][i] * inv;
                const _Float16 h = (_Float16)y;
                qh[j][i] = h;
                // (an infinite query: its difference with itself would be a NaN)
                ql[j][i] = fabsf(y) < INFINITY ? (_Float16)(y - (float)h) : (_Float16)0.f;
            }
    }
    __device__ __forceinline__ void load_k(const _Float16 *head, int kpos, int g)
    {
        const _Float16 *p = head + (size_t)kpos * KV_D + 8 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const half8 *>(p + 32 * j);
    }
    __device__ __forceinline__ void load_v(const _Float16 *head, const int (&vpos)[4], int c)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = *reinterpret_cast<const half8 *>(head + (size_t)vpos[e] * KV_D + 8 * c);
    }
    __device__ __forceinline__ f32x4 scores() const
    {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a = mfma_f16(k[j], qh[j], a);
            b = mfma_f16(k[j], ql[j], b);
        }
        return (a + b) * qscale;
    }
    __device__ __forceinline__ void pv(const f32x4 &p, f32x4 (&acc)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 8; ++x) acc[x] = mfma_f32((float)v[e][x], p[e], acc[x]);
    }
    __device__ __forceinline__ float odd() const
    {
        float z = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 8; ++x) z = fmaf((float)v[e][x], 0.f, z);
        return z;
    }
    static __device__ __forceinline__ int dim(int x, int e, int g) { return 32 * g + 8 * e + x; }
    static __device__ __forceinline__ void put(float *o, const f32x4 (&acc)[8], int g, float s)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                *reinterpret_cast<float4 *>(o + 32 * g + 8 * e + 4 * c) =
                    make_float4(acc[4 * c][e] * s, acc[4 * c + 1][e] * s, acc[4 * c + 2][e] * s,
                                acc[4 * c + 3][e] * s);
    }
};

template <class T>
__global__ __launch_bounds__(64 * FEW_WAVES) void paged_few_kernel(
    PagedKv kv, int few_rows, int max_workers, const float *__restrict__ q, int part_rows,
    float *__restrict__ part, float *__restrict__ out)
{
    extern __shared__ long long before[]; // [seqs + 1]
    __shared__ long long wsum[4];
    const FewPlan plan = few_plan(kv, few_rows, max_workers, before, wsum);
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    // (uniform over the wave, and known to be)
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x * FEW_WAVES + (threadIdx.x >> 6));
    if (w >= plan.workers) return;
    long long at = plan.total * w / plan.workers;
    const long long stop = plan.total * (w + 1) / plan.workers;
    const int rep = kv.heads / kv.kvh;
    const size_t hsize = (size_t)KV_D << kv.shift, psize = 2 * hsize * kv.kvh;
    const int pmask = (1 << kv.shift) - 1;
    const float sc = 1.4426950408889634f * 0.08838834764831845f; // log2(e) / sqrt(128)

    // the slot that holds tile `at`: the last with before[s] <= at
    int s = 0;
    {
        int hi = kv.seqs; // before[hi] > at
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (before[mid] <= at) s = mid;
            else hi = mid;
        }
    }
    while (at < stop) {
        while (before[s + 1] <= at) ++s; // slots without tiles
        const SlotRows sr = slot_rows(kv, s);
        const int tiles = slot_tiles(sr);
        const int in = (int)(at - before[s]);
        const int kh = in / tiles, t0 = in % tiles;
        const int t1 = (int)min((long long)tiles, t0 + (stop - at));
        at += t1 - t0;

        // this lane's row: token c / rep of the slot's new rows
        const int tok = c / rep;
        const bool ok = tok < sr.n;
        const int head = kh * rep + c % rep;
        const size_t row = (size_t)(sr.begin + (ok ? tok : 0)) * kv.heads + head;
        const int first = sr.len - sr.n;           // the first new row's position
        const int sees = ok ? first + tok : -1;    // this row's last visible position
        Ops<T> ops;
        ops.load_q(q + row * KV_D, ok, g);
        f32x4 acc[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        const int *entries = kv.table + (size_t)s * kv.stride;
        const int per = kv.shift - 4; // log2 of a page's tiles
        int have = -64, pages = -1;   // lane i: the slot's page have + i
        auto page_of = [&](int t) {
            const int p = t >> per;
            if (p - have >= 64 || p < have) {
                have = p;
                pages = have + lane < kv.stride ? entries[have + lane] : -1;
            }
            return __builtin_amdgcn_readlane(pages, p - have);
        };
        auto base_of = [&](int page) {
            return (const T *)kv.pages + (size_t)page * psize + (size_t)kh * hsize;
        };
        // positions of a tile, those past the slot's length taken from its
        // last one (a valid row, whose weight is zero)
        auto load = [&](int t, int page, bool keys, bool values) {
            const int p0 = t * FEW_TILE, lim = sr.len - 1 - p0, in_page = p0 & pmask;
            const T *b = base_of(page);
            if (keys) ops.load_k(b, in_page + min(c, lim), g);
            if (values) {
                int vp[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) vp[e] = in_page + min(4 * g + e, lim);
                ops.load_v(b + hsize * kv.kvh, vp, c);
            }
        };
        // tiles whose page the table does not name are not seen
        auto valid = [&](int page) { return sr.len > 0 && (unsigned)page < (unsigned)kv.npages; };
        int page = page_of(t0);
        if (valid(page)) load(t0, page, true, true);
        for (int t = t0; t < t1; ++t) {
            const int next = t + 1 < t1 ? page_of(t + 1) : -1;
            if (!valid(page)) {
                page = next;
                if (valid(page)) load(t + 1, page, true, true);
                continue;
            }
            f32x4 sv = ops.scores();
            if (valid(next)) load(t + 1, next, true, false);
            const int p0 = t * FEW_TILE + 4 * g;
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sv[e] = p0 + e <= sees ? sv[e] * sc : -INFINITY;
                mx = fmaxf(mx, sv[e]);
            }
            mx = wave::max_halves(wave::max_rows2(mx));
            const float mn = fmaxf(m, mx);
            // a row that has seen nothing yet keeps zero weights
            const float base = mn == -INFINITY ? 0.f : mn;
            const float corr = __builtin_amdgcn_exp2f(m - base);
            float rs = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sv[e] = __builtin_amdgcn_exp2f(sv[e] - base);
                rs += sv[e];
            }
            if (__any(mn != m)) {
#pragma unroll
                for (int x = 0; x < 8; ++x) acc[x] *= corr;
                l *= corr;
            }
            l += rs;
            m = mn;
            // a tile that some row sees in part: a value there that is not finite
            // must not reach the rows that do not see it (0 * inf)
            if (t * FEW_TILE + FEW_TILE - 1 > first && __any(ops.odd() != 0.f)) {
                const T *vb = base_of(page) + hsize * kv.kvh;
                for (int i = 0; i < FEW_TILE; ++i) {
                    const int src = (i >> 2) * 16 + c;
                    const float p = i & 2 ? (i & 1 ? __shfl(sv[3], src, 64) : __shfl(sv[2], src, 64))
                                          : (i & 1 ? __shfl(sv[1], src, 64) : __shfl(sv[0], src, 64));
                    if (t * FEW_TILE + i > sees) continue;
                    const T *vr = vb + (size_t)((t * FEW_TILE + i) & pmask) * KV_D;
#pragma unroll
                    for (int x = 0; x < 8; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[x][e] = fmaf(p, (float)vr[Ops<T>::dim(x, e, g)], acc[x][e]);
                }
            } else {
                ops.pv(sv, acc);
            }
            if (valid(next)) load(t + 1, next, false, true);
            page = next;
        }
        l = wave::sum_halves(wave::sum_rows2(l));
        if (t0 == 0 && t1 == tiles) {
            // (a row that saw nothing gives zeros)
            if (ok) Ops<T>::put(out + row * KV_D, acc, g, l > 0.f || l != l ? 1.f / l : 0.f);
        } else if (ok) {
            const long long slot = (long long)w + (long long)s * kv.kvh + kh;
            float *o = part + ((size_t)slot * part_rows + c) * PAGED_PART;
            if (g == 0) {
                o[0] = m;
                o[1] = l;
            }
            Ops<T>::put(o + 4, acc, g, 1.f);
        }
    }
}

// Joins the parts of the units that several workers shared, in worker order.
// Grid (kv heads, seqs), 256 threads: two rows at a time, a dim per thread.
__global__ __launch_bounds__(256) void paged_few_merge_kernel(PagedKv kv, int few_rows,
                                                              int max_workers, int part_rows,
                                                              const float *__restrict__ part,
                                                              float *__restrict__ out)
{
    extern __shared__ long long before[];
    __shared__ long long wsum[4];
    const FewPlan plan = few_plan(kv, few_rows, max_workers, before, wsum);
    const int s = blockIdx.y, kh = blockIdx.x;
    const SlotRows sr = slot_rows(kv, s);
    const int tiles = few_tiles(kv, s, few_rows);
    if (tiles == 0) return;
    const long long first = before[s] + (long long)kh * tiles, last = first + tiles - 1;
    // the worker of tile x: the largest w with total * w / workers <= x
    auto worker = [&](long long x) {
        return (int)(((x + 1) * plan.workers - 1) / plan.total);
    };
    const int w0 = worker(first), w1 = worker(last);
    if (w0 == w1) return; // written whole
    const int rep = kv.heads / kv.kvh;
    const long long slot0 = (long long)w0 + (long long)s * kv.kvh + kh;
    const int d = threadIdx.x & 127;
    for (int c = threadIdx.x >> 7; c < sr.n * rep; c += 2) {
        const float *p = part + ((size_t)slot0 * part_rows + c) * PAGED_PART;
        const size_t step = (size_t)part_rows * PAGED_PART;
        float M = -INFINITY;
        for (int i = 0; i <= w1 - w0; ++i) M = fmaxf(M, p[i * step]);
        const float base = M == -INFINITY ? 0.f : M;
        float num = 0.f, den = 0.f;
        for (int i = 0; i <= w1 - w0; ++i) {
            const float x = __builtin_amdgcn_exp2f(p[i * step] - base);
            den = fmaf(x, p[i * step + 1], den);
            num = fmaf(x, p[i * step + 4 + d], num);
        }
        const size_t row = (size_t)(sr.begin + c / rep) * kv.heads + kh * rep + c % rep;
        out[row * KV_D + d] = den > 0.f || den != den ? num / den : 0.f;
    }
}

constexpr int FEW_MAX_WORKERS = 2048; // eight waves on each of 256 CUs

} // namespace

int paged_few_rows(int rep) { return 16 / rep; }

size_t paged_few_scratch(int seqs, int kvh, int heads, int few)
{
    const int part_rows = few * (heads / kvh);
    return ((size_t)FEW_MAX_WORKERS + (size_t)seqs * kvh) * part_rows * PAGED_PART * 4;
}

int launch_paged_few(const PagedKv &kv, int few, const float *q, float *part, float *out,
                     void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const int part_rows = few * (kv.heads / kv.kvh);
    const size_t lds = ((size_t)kv.seqs + 1) * 8;
    const dim3 grid(FEW_MAX_WORKERS / FEW_WAVES), block(64 * FEW_WAVES);
    if (kv.f16)
        hipLaunchKernelGGL(paged_few_kernel<_Float16>, grid, block, lds, st, kv, few,
                           FEW_MAX_WORKERS, q, part_rows, part, out);
    else
        hipLaunchKernelGGL(paged_few_kernel<float>, grid, block, lds, st, kv, few,
                           FEW_MAX_WORKERS, q, part_rows, part, out);
    hipLaunchKernelGGL(paged_few_merge_kernel, dim3(kv.kvh, kv.seqs), dim3(256), lds, st, kv,
                       few, FEW_MAX_WORKERS, part_rows, part, out);
    return (int)hipGetLastError();
}

} // namespace hyq
