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
// units are numbered in order and each of W workers takes the next T / W of
// them. A range that covers a unit whole writes the output,
// a part of one its maximum, sum and unnormalised row to slot w + u (workers
// and units both ascend, so w + u names each pair once), which the merge
// joins in worker order. The worker of a unit's first tile notes who shares it.
//
// Bound by memory, and for few positions by the loads that wait for each other
// (starts and lengths, table, keys) and the merge's launch. With the merge: 64
// slots of up to 8192 positions, 32 heads over 8, f16 pages, 143 us for 848 MB
// (5.9 TB/s; with 32 positions a step 149, with 64 153); four of up to 60001, 16 over 4, f32 pages, 105 us for 642 MB (6.1);
// two of up to 1100, 11.8 us, of which the merge's launch takes 4.4.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "hyq_paged_attn.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int FEW_WAVES = 4;
constexpr int TILE = 16; // positions of a step

// Worker w of `workers` takes `base` tiles, the first `more` workers one more.
struct FewPlan {
    long long total;
    int workers, base, more;
    __device__ __forceinline__ long long begin(int w) const
    {
        return (long long)w * base + min(w, more);
    }
    // the worker that takes tile x
    __device__ __forceinline__ int worker(long long x) const
    {
        const long long longer = (long long)more * (base + 1);
        return x < longer ? divide(x, base + 1) : more + divide(x - longer, base);
    }
};

// (new rows over no positions still have their zeros to be written: one tile)
__device__ __forceinline__ int slot_tiles(const SlotRows &r)
{
    return max(1, (r.len + TILE - 1) / TILE);
}
__device__ __forceinline__ int few_tiles(const PagedKv &kv, int s, int few_rows)
{
    const SlotRows r = slot_rows(kv, s);
    return r.n > 0 && r.n <= few_rows ? slot_tiles(r) : 0;
}

// before[s], in LDS: the tiles of the slots before s over all KV heads, with
// the total at before[seqs]. 256 threads. (Every workgroup forms it for itself:
// a launch before this one would cost more than the few loads and barriers.)
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
    // (a tile for a worker, while there are fewer tiles than workers: two slots of
    // 1100 positions in f32 pages 11.8 us, two tiles a worker 13.0)
    p.workers = (int)min((long long)max_workers, carry);
    p.base = divide(carry, max(p.workers, 1));
    p.more = (int)(carry - (long long)p.base * p.workers);
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

// A vector of the cache: ONCE, of pages that one slot reads, not to be kept in the
// caches, which the rows and parts of this launch and the next ones are for.
template <class V, bool ONCE, class T>
__device__ __forceinline__ V cached(const T *base, unsigned off)
{
    const V *p = reinterpret_cast<const V *>(reinterpret_cast<const char *>(base) +
                                             (unsigned)(off * sizeof(T)));
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}

// The operands of one tile, by element type. Dims of an output element
// acc[x][e] (see pv): f32 64 (x / 4) + 16 g + 4 e + x % 4, f16 32 g + 8 e + x.
template <class T> struct Ops;

template <> struct Ops<float> {
    float4 q[8]; // row lane % 16, dims 16 j + 4 g ..
    f32x4 k[8];  // position lane % 16, the same dims
    f32x4 v[8];  // position 4 g + x / 2, dims 64 (x % 2) + 4 (lane % 16) ..
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
    template <bool ONCE>
    __device__ __forceinline__ void load_k(const float *head, int kpos, int g)
    {
        const unsigned o = kpos * KV_D + 4 * g;
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = cached<f32x4, ONCE>(head, o + 16 * j);
    }
    template <bool ONCE>
    __device__ __forceinline__ void load_v(const float *head, const int (&vpos)[4], int c)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned o = vpos[e] * KV_D + 4 * c;
            v[2 * e] = cached<f32x4, ONCE>(head, o);
            v[2 * e + 1] = cached<f32x4, ONCE>(head, o + 64);
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
                const f32x4 x = v[2 * e + c];
                acc[4 * c] = mfma_f32(x.x, p[e], acc[4 * c]);
                acc[4 * c + 1] = mfma_f32(x.y, p[e], acc[4 * c + 1]);
                acc[4 * c + 2] = mfma_f32(x.z, p[e], acc[4 * c + 2]);
                acc[4 * c + 3] = mfma_f32(x.w, p[e], acc[4 * c + 3]);
            }
    }
    // values that are not finite become zero; whether the wave had any
    __device__ __forceinline__ bool clean()
    {
        float z = 0.f; // (a sum of v * 0: not zero if one is not finite)
#pragma unroll
        for (int x = 0; x < 8; ++x)
            z = fmaf(v[x].x, 0.f,
                     fmaf(v[x].y, 0.f, fmaf(v[x].z, 0.f, fmaf(v[x].w, 0.f, z))));
        if (!__any(z != 0.f)) return false;
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[x][i] = fabsf(v[x][i]) < INFINITY ? v[x][i] : 0.f;
        return true;
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
        const int e = query_exponent(mx);
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
    template <bool ONCE>
    __device__ __forceinline__ void load_k(const _Float16 *head, int kpos, int g)
    {
        const unsigned o = kpos * KV_D + 8 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = cached<half8, ONCE>(head, o + 32 * j);
    }
    template <bool ONCE>
    __device__ __forceinline__ void load_v(const _Float16 *head, const int (&vpos)[4], int c)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = cached<half8, ONCE>(head, vpos[e] * KV_D + 8 * c);
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
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int x = 0; x < 8; ++x) acc[x] = mfma_f32((float)v[e][x], p[e], acc[x]);
            // (keeps the widened values of later positions out of registers)
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __device__ __forceinline__ bool clean()
    {
        half8 z = {}; // (a sum of v * 0)
#pragma unroll
        for (int e = 0; e < 4; ++e) z += v[e] * (_Float16)0.f;
        const u32x4 w = __builtin_bit_cast(u32x4, z); // (a NaN, or zeros of any sign)
        if (!__any(((w[0] | w[1] | w[2] | w[3]) & 0x7fff7fffu) != 0)) return false;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) { // (two f16 of exponent all ones or not)
                u32x4 w = __builtin_bit_cast(u32x4, v[e]);
                w[x] = (w[x] & 0x7c00u) == 0x7c00u ? w[x] & 0xffff0000u : w[x];
                w[x] = (w[x] & 0x7c000000u) == 0x7c000000u ? w[x] & 0x0000ffffu : w[x];
                v[e] = __builtin_bit_cast(half8, w);
            }
        return true;
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
__global__ __launch_bounds__(64 * FEW_WAVES, 2) void paged_few_kernel(
    PagedKv kv, int few_rows, int max_workers, RowsScratch rs, const float *__restrict__ q,
    int part_rows, float *__restrict__ part, int2 *__restrict__ shared, float *__restrict__ out)
{
    extern __shared__ long long before[]; // [seqs + 1]
    __shared__ long long wsum[4];
    if (blockIdx.x * FEW_WAVES >= max_workers) { // one more workgroup: the tile form's plan
        rows_plan(kv, few_rows, rs, (int *)before);
        return;
    }
    const FewPlan plan = few_plan(kv, few_rows, max_workers, before, wsum);
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    // (uniform over the wave, and known to be; few workers lie on many CUs: two
    // slots of 1100 positions took 1.5 us longer with four to a workgroup)
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x + max_workers / FEW_WAVES *
                                                                  (threadIdx.x >> 6));
    if (w >= plan.workers) return;
    long long at = plan.begin(w);
    const long long stop = plan.begin(w + 1);
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
        s = __builtin_amdgcn_readfirstlane(s); // (what comes from LDS, known to be uniform)
        const SlotRows sr = slot_rows(kv, s);
        const int tiles = slot_tiles(sr);
        const int in = __builtin_amdgcn_readfirstlane((int)(at - before[s]));
        const int kh = in / tiles, t0 = in % tiles;
        const int t1 = __builtin_amdgcn_readfirstlane(
            (int)min((long long)tiles, t0 + (stop - at)));
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
        int have = -64, pages = -1; // lane i: the slot's page have + i
        // the page of 16 positions, -1 where the slot has none
        auto page_of = [&](int p0) {
            const int p = p0 >> kv.shift;
            if (p - have >= 64 || p < have) {
                have = p;
                pages = have + lane < kv.stride ? entries[have + lane] : -1;
            }
            const int id = __builtin_amdgcn_readlane(pages, p - have);
            return p0 < sr.len && (unsigned)id < (unsigned)kv.npages ? id : -1;
        };
        // A step's loads are unconditional: positions past the length are taken
        // from the last one, and where there is no page from the pool's first
        // (their weights are zero, and values that are not finite are cleared).
        auto head_of = [&](int page) {
            return (const T *)kv.pages + (size_t)max(page, 0) * psize + (size_t)kh * hsize;
        };
        auto load_k = [&](auto once, int p, int page) {
            ops.template load_k<once.value>(
                head_of(page), (p & pmask) + max(min(c, sr.len - 1 - p), 0), g);
        };
        auto load_v = [&](auto once, int p, int page) {
            int vp[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                vp[e] = (p & pmask) + max(min(4 * g + e, sr.len - 1 - p), 0);
            ops.template load_v<once.value>(head_of(page) + hsize * kv.kvh, vp, c);
        };
        // Whether the range begins in a page that neither neighbouring slot names
        // at this place: beams of one prompt share their pages, and find them in
        // the caches. Read as such and as read once, us for 64 slots of up to 8192
        // positions: 167 and 147 where none share, 131 and 152 where fours do.
        const int at0 = min((t0 * TILE) >> kv.shift, kv.stride - 1);
        const int mine = entries[at0], below = s ? entries[at0 - kv.stride] : -1,
                  above = s + 1 < kv.seqs ? entries[at0 + kv.stride] : -1;
        int page = page_of(t0 * TILE);
        const bool alone =
            __builtin_amdgcn_readfirstlane(mine != below && mine != above) != 0;
        bool odd = false;
        auto stream = [&](auto once) {
            load_k(once, t0 * TILE, page);
            load_v(once, t0 * TILE, page);
            for (int t = t0; t < t1; ++t) {
                const int p0 = t * TILE, pn = min(t + 1, t1 - 1) * TILE;
                f32x4 sv = ops.scores();
                const int next = page_of(pn);
                load_k(once, pn, next);
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool see = p0 + 4 * g + e <= sees && page >= 0;
                    sv[e] = see ? sv[e] * sc : -INFINITY;
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
                // a step that some row does not see whole: a value that is not finite
                // must not reach the rows that do not see it (0 * inf), see below
                if (p0 + TILE - 1 > first || page < 0) odd |= ops.clean();
                ops.pv(sv, acc);
                load_v(once, pn, next);
                page = next;
            }
        };
        if (alone) stream(std::true_type{});
        else stream(std::false_type{});
        if (odd) {
            // the values left out of the steps above, for the rows that see
            // them: whatever its weight, such a value makes the sum not finite
            for (int p = t0 * TILE; p < min(t1 * TILE, sr.len); ++p) {
                const int id = page_of(p & ~15);
                if ((p | 15) <= first || id < 0 || p > sees) continue;
                const T *vr = head_of(id) + hsize * kv.kvh + (p & pmask) * KV_D;
#pragma unroll
                for (int x = 0; x < 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = (float)vr[Ops<T>::dim(x, e, g)];
                        acc[x][e] += fabsf(y) < INFINITY ? 0.f : y;
                    }
            }
        }
        l = wave::sum_halves(wave::sum_rows2(l));
        if (t0 == 0 && lane == 0) { // who shares the unit, for the merge
            const long long last = before[s] + (long long)(kh + 1) * tiles - 1;
            const int n = t1 == tiles ? 1 : plan.worker(last) - w + 1;
            shared[(size_t)s * kv.kvh + kh] = make_int2(w, n);
        }
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

// ROWS rows' parts p, p + step, ..., n of each, eight in flight in all: the
// running maxima m, exp-sums l and a lane's sums x.
template <class V, int ROWS> struct Joined {
    float m[ROWS], l[ROWS];
    V x[ROWS];
    __device__ __forceinline__ Joined()
    {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
            x[r] = V{};
        }
    }
    __device__ __forceinline__ void add(const float *const (&p)[ROWS], size_t step, int n, int d)
    {
        constexpr int DEPTH = 8 / ROWS;
        for (int b = 0; b < n; b += DEPTH) {
            float2v ml[ROWS][DEPTH];
            V v[ROWS][DEPTH];
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int k = 0; k < DEPTH; ++k) {
                    const float *o = p[r] + (size_t)min(b + k, n - 1) * step;
                    ml[r][k] = *reinterpret_cast<const float2v *>(o);
                    v[r][k] = *reinterpret_cast<const V *>(o + 4 + d);
                }
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                float top = m[r];
#pragma unroll
                for (int k = 0; k < DEPTH; ++k) top = fmaxf(top, ml[r][k][0]);
                const float base = top == -INFINITY ? 0.f : top;
                const float c = __builtin_amdgcn_exp2f(m[r] - base);
                l[r] *= c;
                x[r] *= c;
                m[r] = top;
#pragma unroll
                for (int k = 0; k < DEPTH; ++k) {
                    const float w = b + k < n ? __builtin_amdgcn_exp2f(ml[r][k][0] - base) : 0.f;
                    l[r] = fmaf(w, ml[r][k][1], l[r]);
                    x[r] += w * v[r][k];
                }
            }
        }
    }
    // what a row's sums are to be multiplied with (a row that saw nothing: 0)
    __device__ __forceinline__ float scale(int r) const
    {
        return l[r] > 0.f || l[r] != l[r] ? 1.f / l[r] : 0.f;
    }
};

// Joins the parts of a slot's rows over a KV head, where several workers shared
// them, by 256 threads, lane d dims 2 d and 2 d + 1. wide: row c by all four
// waves, a quarter of the parts each, joined in wave order; otherwise rows c ..
// c + 3, one per wave.
__device__ __forceinline__ void merge_few(const PagedKv &kv, int few_rows, int part_rows,
                                          const float *__restrict__ part,
                                          const int2 *__restrict__ shared, float *__restrict__ out,
                                          int kh, int s, int c, bool wide)
{
    __shared__ float red[4][KV_D + 2];
    const int rep = kv.heads / kv.kvh;
    const int2 by = shared[(size_t)s * kv.kvh + kh]; // (of a slot without rows: anything)
    const SlotRows sr = slot_rows(kv, s);
    if (sr.n > few_rows || c >= sr.n * rep) return;
    const int w0 = by.x, n = by.y;
    if (n == 1) return; // written whole
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int r = wide ? c : c + g;
    if (!wide && r >= sr.n * rep) return;
    const size_t step = (size_t)part_rows * PAGED_PART;
    const float *p = part + ((size_t)((long long)w0 + (long long)s * kv.kvh + kh) * part_rows + r) *
                                PAGED_PART;
    const int a = wide ? n * g / 4 : 0, b = wide ? n * (g + 1) / 4 : n;
    Joined<float2v, 1> j;
    j.add({p + (size_t)a * step}, step, b - a, 2 * lane);
    float *o = out + ((size_t)(sr.begin + r / rep) * kv.heads + kh * rep + r % rep) * KV_D;
    if (!wide) {
        *reinterpret_cast<float2v *>(o + 2 * lane) = j.x[0] * j.scale(0);
        return;
    }
    red[g][2 * lane] = j.x[0][0];
    red[g][2 * lane + 1] = j.x[0][1];
    if (lane == 0) {
        red[g][KV_D] = j.m[0];
        red[g][KV_D + 1] = j.l[0];
    }
    __syncthreads();
    if (g) return;
    const float M = fmaxf(fmaxf(red[0][KV_D], red[1][KV_D]), fmaxf(red[2][KV_D], red[3][KV_D]));
    const float base = M == -INFINITY ? 0.f : M;
    j.l[0] = 0.f;
    j.x[0] = float2v{0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(red[w][KV_D] - base);
        j.l[0] = fmaf(f, red[w][KV_D + 1], j.l[0]);
        j.x[0] += f * float2v{red[w][2 * lane], red[w][2 * lane + 1]};
    }
    *reinterpret_cast<float2v *>(o + 2 * lane) = j.x[0] * j.scale(0);
}

// Joins the pieces of a block that was cut, by 256 threads: MERGE_ROWS rows, two
// for a 32-lane half wave, lane d dims 4 d ..
__device__ __forceinline__ void merge_rows(const PagedKv &kv, const RowsScratch &rs,
                                           float *__restrict__ out, int kh, int b, int part)
{
    const Block blk = rs.blocks[b];
    if (b >= rs.plan->blocks || blk.pieces < 2) return;
    const int rep = kv.heads / kv.kvh;
    const int r = part * MERGE_ROWS + (threadIdx.x >> 5), d = 4 * (threadIdx.x & 31);
    if (r / rep >= blk.toks) return;
    const float *p = rs.parts + (((size_t)blk.part * kv.kvh + kh) * PR_ROWS + r) * PAGED_PART;
    Joined<f32x4, 2> j; // (a row past the block's is not stored)
    j.add({p, p + 8 * PAGED_PART}, (size_t)kv.kvh * PR_ROWS * PAGED_PART, blk.pieces, d);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int at = r + 8 * i, tl = at / rep;
        if (tl < blk.toks)
            *reinterpret_cast<f32x4 *>(
                out + ((size_t)(blk.row + tl) * kv.heads + kh * rep + at % rep) * KV_D + d) =
                j.x[i] * j.scale(i);
    }
}

// Grid: the slots' rows, one or four a workgroup, then the blocks', MERGE_ROWS a
// workgroup; the KV heads of a row in sequence.
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedKv kv, int few_rows, int part_rows,
                                                          int wide, RowsScratch rs,
                                                          const float *__restrict__ part,
                                                          const int2 *__restrict__ shared,
                                                          float *__restrict__ out)
{
    const int each = wide ? part_rows : (part_rows + 3) / 4; // workgroups of a slot and KV head
    const int kh = blockIdx.x % kv.kvh, i = blockIdx.x / kv.kvh, n = kv.seqs * each;
    if (i < n)
        merge_few(kv, few_rows, part_rows, part, shared, out, kh, i / each,
                  (i % each) * (wide ? 1 : 4), wide != 0);
    else
        merge_rows(kv, rs, out, kh, (i - n) / (PR_ROWS / MERGE_ROWS),
                   (i - n) % (PR_ROWS / MERGE_ROWS));
}

// Workers: a wave on each SIMD for f32 pages, two for f16 pages, whose steps
// have twice the products for each byte (64 sessions of up to 8192 positions in
// f16 pages: 184 us with 1024, 143 with 2048, 149 with 3072; four of up to 60001
// in f32 pages: 105 with 1024, 113 with 2048). Numbers between leave SIMDs
// unequal: 165 with 1536 in f16 pages, 146 with 1280 in f32 ones.
int few_workers(bool f16) { return f16 ? 2048 : 1024; }

} // namespace

// The rows of one tile. (Where a slot has more, the rows' form: 32 slots of up to
// 4000 positions, 16 heads over 4, took 43 us here with four new tokens each in
// f16 pages and 48 in f32 ones, with five 45 and 60 there; here the positions
// would be read twice.)
int paged_few_rows(int rep) { return 16 / rep; }

namespace {

size_t parts_bytes(bool f16, int seqs, int kvh, int part_rows)
{
    return ((size_t)few_workers(f16) + (size_t)seqs * kvh) * part_rows * PAGED_PART * 4;
}

} // namespace

// Parts, then the workers of each slot and KV head.
size_t paged_few_scratch(bool f16, int seqs, int kvh, int heads, int few)
{
    const size_t shared = ((size_t)seqs * kvh * 8 + 255) / 256 * 256;
    return parts_bytes(f16, seqs, kvh, few * (heads / kvh)) + shared;
}

int launch_paged_few(const PagedKv &kv, int few, const RowsScratch &rs, const float *q, float *part,
                     float *out, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const int part_rows = few * (kv.heads / kv.kvh);
    int2 *shared = (int2 *)((char *)part + parts_bytes(kv.f16, kv.seqs, kv.kvh, part_rows));
    const size_t lds = ((size_t)kv.seqs + 1) * 8;
    const int workers = few_workers(kv.f16);
    const dim3 grid(workers / FEW_WAVES + (rs.cap > 0)), block(64 * FEW_WAVES);
    if (kv.f16)
        hipLaunchKernelGGL(paged_few_kernel<_Float16>, grid, block, lds, st, kv, few, workers, rs, q,
                           part_rows, part, shared, out);
    else
        hipLaunchKernelGGL(paged_few_kernel<float>, grid, block, lds, st, kv, few, workers, rs, q,
                           part_rows, part, shared, out);
    return (int)hipGetLastError();
}

int launch_paged_merge(const PagedKv &kv, int few, const RowsScratch &rs, const float *part,
                       float *out, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const int part_rows = few * (kv.heads / kv.kvh);
    const int2 *shared =
        (const int2 *)((const char *)part + parts_bytes(kv.f16, kv.seqs, kv.kvh, part_rows));
    // Few rows have many parts each (1024 workers over four slots of four KV
    // heads: 64), which all of a workgroup's waves read; many rows have few, and
    // a wave each. Wide and not: four slots of 60001 positions 124 and 134 us,
    // 64 slots of 8192 173 and 170.
    const int wide = kv.seqs * kv.kvh * part_rows <= 1024;
    const int each = wide ? part_rows : (part_rows + 3) / 4;
    const dim3 grid((unsigned)merge_groups(kv.seqs, kv.kvh, each, rs.cap));
    hipLaunchKernelGGL(paged_merge_kernel, grid, dim3(256), 0, st, kv, few, part_rows, wide, rs, part,
                       shared, out);
    return (int)hipGetLastError();
}

} // namespace hyq
