// Attention over a paged cache for slots of many new rows (prompts): causal,
// on the matrix cores, for a ragged batch.
//
// A workgroup takes the query rows of one KV head for a block of a slot's new
// tokens - 128 rows, row r = token r / rep of the block, query head r % rep of
// the group - and a range of 64-position steps. Wave w owns rows 32 (w % 4) ..
// and of every step the 32 positions of its half w / 4; it forms transposed
// products with v_mfma_f32_32x32x16_f16, so that a lane holds one query row
// (lane % 32) and 16 of its positions or dims:
//   S^T [32 pos x 32 rows]   = K . Q^T, lane (c, h): positions 8a + 4h + b
//   O^T [128 dims x 32 rows] += V^T . P^T
// with the softmax's running maximum and sum per lane (one exchange between
// the row's two lanes). The second product takes its positions in the order in
// which the lane holds them, so no weight moves between lanes. An f32 operand x
// is split into f16 parts hi = f16(x), lo = f16(x - hi) and products sum
// hi.hi + lo.hi + hi.lo in f32, which keeps the scores and sums near f32
// accuracy; f16 pages are exact as they are and need no low parts of keys and
// values. f32 pages hold keys and values below 65504, of which those from 2^-14
// up keep 22 bits.
//
// Keys and values go through LDS, two steps of them, rows as they are (values
// are transposed by ds_read_b64_tr_b16 on their way to the matrix operand).
// The next step is converted and stored between the products of the present
// one, and the step after it loaded, with one barrier a step.
//
// Blocks of different slots and places see very different numbers of steps, so
// a plan cuts them (rows_plan): one workgroup counts every block's steps and
// makes pieces of about equal length, enough to fill the GPU once, and the
// pieces of a block that was cut leave partial rows, which a merge joins in
// order.
//
// Bound by a step's matrix products (1.8 us at the rate at which all SIMDs
// sustain them for f32 pages, 1.2 for f16), its LDS traffic (0.6) and its VALU
// work, which overlap in part: a step takes 3.0 and 1.8 us. 512 new tokens of
// one slot over 2012 positions, 16 heads over 4, f32 pages: 45 us in all, the
// plan 6, this launch 37 (eight steps, and 13 us to begin and end: cold code and
// loads that wait for each other), the merge 5.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged_attn.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float float2v __attribute__((ext_vector_type(2)));

constexpr int PR_THREADS = 512;     // two waves on each SIMD
// Row pitches in halves, chosen for the banks: keys are read 16 bytes a lane
// from 16 rows (4 banks apart), values by the transposing read 8 bytes a lane
// from 4 rows (16 banks apart).
constexpr int PR_KP = KV_D + 8;
constexpr int PR_VP = KV_D + 32;

__device__ __forceinline__ f32x16 mfma(const half8 &a, const half8 &b, const f32x16 &c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// Two values' high and low f16 parts, both rounded to nearest: hi, and
// x - hi (exact in f32) by one mixed-precision fma each.
__device__ __forceinline__ void split2(float x, float y, half2 &hi, half2 &lo)
{
    hi = __builtin_convertvector((float2v{x, y}), half2);
    float a, b;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(hi), "v"(x));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(b)
        : "v"(hi), "v"(y));
    lo = __builtin_convertvector((float2v{a, b}), half2);
}
// The same with the low parts 2^11 times as large: an operand keeps 22 bits as
// long as its high part is a normal number (from 2^-14 up), where low parts in
// place would be subnormal below 2^-3. The factor is taken off the scores' sum
// of such products, and off the weights that values' low parts are multiplied
// with.
constexpr float LO_SCALE = 2048.f;
__device__ __forceinline__ void split2_scaled(float x, float y, half2 &hi, half2 &lo)
{
    hi = __builtin_convertvector((float2v{x, y}), half2);
    float a, b;
    asm("v_fma_mix_f32 %0, -%1, %3, %2 op_sel_hi:[1,0,0]"
        : "=v"(a)
        : "v"(hi), "v"(x * LO_SCALE), "s"(LO_SCALE));
    asm("v_fma_mix_f32 %0, -%1, %3, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(b)
        : "v"(hi), "v"(y * LO_SCALE), "s"(LO_SCALE));
    lo = __builtin_convertvector((float2v{a, b}), half2);
}
// Positions p .. p + 3 of 16 dims: lane i of 16 takes dim i of them all, its
// address being that of row (i / 4), dims 4 (i % 4) ..
__device__ __forceinline__ half4 read_transposed(const _Float16 *p)
{
    typedef short short4v __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(
        half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) short4v *)const_cast<_Float16 *>(p)));
}

// Whether f16 parts hold a value: from 65520 on the high one would be infinite.
// (Any finite f16 does.)
__device__ __forceinline__ bool has_parts(float x) { return fabsf(x) < 65520.f; }

// A step's keys and values on their way from memory to LDS: 512 threads, rows
// of 16 bytes a lane.
template <class T> struct Raw;
template <> struct Raw<float> { // row (t / 32) + 16 i, dims 4 (t % 32) ..
    static constexpr int N = 4;
    typedef float4 Vec;
    Vec k[N], v[N];
    static constexpr int STEP = 16;
    static __device__ __forceinline__ int row(int t) { return t >> 5; }
    static __device__ __forceinline__ int group(int, int i) { return i; } // its 16 rows
    static __device__ __forceinline__ int dim(int t) { return 4 * (t & 31); }
    // values of rows that nobody sees become zero, and those of no f16 parts;
    // whether there were any of the latter in the other rows
    __device__ __forceinline__ bool clean(const bool (&unseen)[N])
    {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            auto one = [&](float &x) {
                const bool fine = has_parts(x);
                odd |= !fine && !unseen[i];
                x = fine && !unseen[i] ? x : 0.f;
            };
            one(v[i].x), one(v[i].y), one(v[i].z), one(v[i].w);
        }
        return odd;
    }
    static __device__ __forceinline__ void put(_Float16 *hi, _Float16 *lo, const float4 &x)
    {
        half2 a, b, c, d;
        split2_scaled(x.x, x.y, a, b);
        split2_scaled(x.z, x.w, c, d);
        *reinterpret_cast<half4 *>(hi) = half4{a[0], a[1], c[0], c[1]};
        *reinterpret_cast<half4 *>(lo) = half4{b[0], b[1], d[0], d[1]};
    }
};
template <> struct Raw<_Float16> { // row (t / 16) + 32 i, dims 8 (t % 16) ..
    static constexpr int N = 2;
    typedef half8 Vec;
    Vec k[N], v[N];
    static constexpr int STEP = 32;
    static __device__ __forceinline__ int row(int t) { return t >> 4; }
    static __device__ __forceinline__ int group(int wave, int i) { return 2 * i + (wave >> 2); }
    static __device__ __forceinline__ int dim(int t) { return 8 * (t & 15); }
    __device__ __forceinline__ bool clean(const bool (&unseen)[N])
    {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool fine = has_parts((float)v[i][e]);
                odd |= !fine && !unseen[i];
                v[i][e] = fine && !unseen[i] ? v[i][e] : (_Float16)0.f;
            }
        return odd;
    }
    static __device__ __forceinline__ void put(_Float16 *hi, _Float16 *, const half8 &x)
    {
        *reinterpret_cast<half8 *>(hi) = x;
    }
};

template <bool LO> struct RowsLds { // one step
    _Float16 khi[PR_TILE][PR_KP], klo[LO ? PR_TILE : 1][PR_KP];
    _Float16 vhi[PR_TILE][PR_VP], vlo[LO ? PR_TILE : 1][PR_VP];
};

// WHOLE: a step lies in one page (of 64 tokens or more), so that it takes one
// look at the table and one base address instead of four of each, whose scalar
// work was a sixth of a wave's time (512 tokens over 32012 positions, pages of 16
// and of 64 tokens: 405 and 394 us in f32 pages, 266 and 249 in f16).
template <class T, bool WHOLE>
__global__ __launch_bounds__(PR_THREADS, 2) void paged_rows_kernel(
    PagedKv kv, RowsScratch rs, const float *__restrict__ q, float *__restrict__ out)
{
    constexpr bool LO = sizeof(T) == 4; // low parts of keys and values
    typedef Raw<T> R;
    constexpr int JOIN = 66; // a lane's words in the join of the two halves
    __shared__ __align__(16) union {
        RowsLds<LO> step[2];
        float join[4][JOIN][64];
    } lds;
    // (a group's KV heads in sequence, so that an XCD, which takes every eighth
    // workgroup, reads few heads' keys and values into its L2)
    const int kh = blockIdx.x % kv.kvh, group = blockIdx.x / kv.kvh;
    const int from = rs.groups[group], to = rs.groups[group + 1]; // (read whatever their number)
    if (group >= rs.plan->groups) return;
#pragma unroll 1
    for (int at_piece = from; at_piece < to; ++at_piece) {
        if (at_piece > from) __syncthreads(); // the last piece's readers of LDS are done
        const Piece piece = rs.pieces[at_piece];
        const int s = piece.slot, tq = rs.tq;
        const int t = threadIdx.x, lane = t & 63, h = lane >> 5, c = lane & 31;
        const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
        const int part_of = wave >> 2, rows = wave & 3;
        const int rep = kv.heads / kv.kvh;
        const size_t hsize = (size_t)KV_D << kv.shift, psize = 2 * hsize * kv.kvh;
        const int pmask = (1 << kv.shift) - 1;
        const float sc = 1.4426950408889634f * 0.08838834764831845f; // log2(e) / sqrt(128)

        const int tok0 = piece.index * tq;
        const int first = piece.first; // position of the slot's first new row
        const int toks = min(tq, piece.n - tok0);
        const int seen_end = first + tok0 + toks; // one past the last position that a row sees
        const int p_end = min(piece.t1 * PR_TILE, seen_end);
        const int p_begin = piece.t0 * PR_TILE;
        const int all_see = first + tok0; // the last position that every row sees

        // The pages of a step's four 16-position groups (or the step's one), -1 where
        // none. Page ids come 64 at a time, one per lane. Rows past the end are
        // loaded too, from the same page or, where there is none, from the pool's
        // first: their weights are zero, and their values, whatever lies there,
        // are cleared.
        const int *entries = kv.table + (size_t)s * kv.stride;
        int have = -64, ids = -1; // lane i: the slot's page have + i
        constexpr int GROUPS = WHOLE ? 1 : 4;
        struct Pages {
            int e[GROUPS];
            __device__ __forceinline__ int of(int group) const { return e[WHOLE ? 0 : group]; }
            __device__ __forceinline__ int at(int g) const // (no index that is not constant)
            {
                return g == 0 ? of(0) : g == 1 ? of(1) : g == 2 ? of(2) : of(3);
            }
            __device__ __forceinline__ bool missing() const
            {
                int all = e[0];
#pragma unroll
                for (int i = 1; i < GROUPS; ++i) all |= e[i];
                return all < 0;
            }
        };
        auto pages_of = [&](int p0) {
            Pages f;
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                const int at = p0 + 16 * i, p = at >> kv.shift;
                if (p - have >= 64 || p < have) {
                    have = p;
                    ids = entries[min(have + lane, kv.stride - 1)];
                }
                const int e = __builtin_amdgcn_readlane(ids, p - have);
                f.e[i] = (WHOLE || at < p_end) && (unsigned)e < (unsigned)kv.npages ? e : -1;
            }
            return f;
        };
        R raw;
        auto load = [&](int p0, const Pages &pg) {
            if constexpr (WHOLE) {
                const T *b = (const T *)kv.pages + (size_t)max(pg.e[0], 0) * psize +
                             (size_t)kh * hsize + (size_t)(p0 & pmask) * KV_D;
#pragma unroll
                for (int i = 0; i < R::N; ++i) {
                    const unsigned o = (R::row(t) + R::STEP * i) * KV_D + R::dim(t);
                    raw.k[i] = at<typename R::Vec>(b, o);
                    raw.v[i] = at<typename R::Vec>(b + hsize * kv.kvh, o);
                }
            } else {
#pragma unroll
                for (int i = 0; i < R::N; ++i) {
                    const int g = R::group(wave, i), e = pg.at(g);
                    // (a uniform base, and an offset that never changes)
                    const T *b = (const T *)kv.pages + (size_t)max(e, 0) * psize +
                                 (size_t)kh * hsize + (size_t)((p0 + 16 * g) & pmask) * KV_D;
                    const unsigned o = (R::row(t) & 15) * KV_D + R::dim(t);
                    raw.k[i] = at<typename R::Vec>(b, o);
                    raw.v[i] = at<typename R::Vec>(b + hsize * kv.kvh, o);
                }
            }
        };
        // one of the 2 N rows of `raw`, converted, to a buffer
        auto store = [&](int buf, int n) {
            RowsLds<LO> &l = lds.step[buf];
            const int d = R::dim(t), r = R::row(t) + R::STEP * (n >> 1);
            if (n & 1)
                R::put(&l.vhi[r][d], &l.vlo[LO ? r : 0][LO ? d : 0], raw.v[n >> 1]);
            else
                R::put(&l.khi[r][d], &l.klo[LO ? r : 0][LO ? d : 0], raw.k[n >> 1]);
        };
        // whether some row sees a step in part
        auto partial = [&](int p0, const Pages &pg) {
            return p0 + PR_TILE - 1 > all_see || pg.missing();
        };
        // `raw` of such a step, cleaned: its rows behind the last one that a query
        // sees, or without a page, may hold anything
        auto clean = [&](int p0, const Pages &pg) {
            bool unseen[R::N];
#pragma unroll
            for (int i = 0; i < R::N; ++i) {
                const int seen = pg.at(R::group(wave, i)) < 0 ? 0 : seen_end - p0 - R::STEP * i;
                unseen[i] = R::row(t) >= seen;
            }
            return raw.clean(unseen);
        };

        Pages cur = pages_of(p_begin), next = pages_of(p_begin + PR_TILE);
        load(p_begin, cur);

        // this lane's query row
        const int r = 32 * rows + c, tl = r / rep;
        const bool ok = tl < toks;
        const int head = kh * rep + r % rep;
        const int sees = ok ? first + tok0 + tl : -1; // its last visible position
        // the last position that the wave's first row sees, and with it all of them
        const int wave_all = first + tok0 + min(toks - 1, (32 * rows) / rep);
        const size_t row = (size_t)(piece.begin + tok0 + (ok ? tl : 0)) * kv.heads + head;

        // q = 2^e (hi + lo), the row's power of two bringing it inside f16's range: to
        // below 2^14 where the low parts stay as they are, and to below 2 where they
        // are scaled like those of the keys that they are added up with.
        half8 qhi[KV_D / 16], qlo[KV_D / 16];
        float qscale;
        {
            // (loaded whatever the row, so that all loads are in flight at once)
            const float *qr = q + row * KV_D + 8 * h;
            float4 x[KV_D / 8];
#pragma unroll
            for (int kk = 0; kk < KV_D / 16; ++kk) {
                x[2 * kk] = *reinterpret_cast<const float4 *>(qr + 16 * kk);
                x[2 * kk + 1] = *reinterpret_cast<const float4 *>(qr + 16 * kk + 4);
            }
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < KV_D / 8; ++k)
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)),
                                     fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
            mx = wave::max_halves(mx);
            const int e = query_exponent(mx) - (LO ? 0 : 13);
            qscale = ldexpf(sc, e);
            const float inv = ok ? ldexpf(1.f, -e) : 0.f;
#pragma unroll
            for (int kk = 0; kk < KV_D / 16; ++kk) {
                const float4 a = x[2 * kk], b = x[2 * kk + 1];
                const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    half2 hi, lo;
                    if constexpr (LO) split2_scaled(v[i] * inv, v[i + 1] * inv, hi, lo);
                    else split2(v[i] * inv, v[i + 1] * inv, hi, lo);
                    qhi[kk][i] = hi[0];
                    qhi[kk][i + 1] = hi[1];
                    qlo[kk][i] = lo[0];
                    qlo[kk][i + 1] = lo[1];
                }
            }
        }

        f32x16 acc[KV_D / 32];
#pragma unroll
        for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
        float m_run = -INFINITY, l_run = 0.f;

        // A step that some row sees in part: values of it that are not finite, or
        // would not be as f16 parts, must not reach the rows that do not see them
        // (0 * inf), see below.
        bool odd = partial(p_begin, cur) && clean(p_begin, cur);
#pragma unroll
        for (int n = 0; n < 2 * R::N; ++n) store(0, n);
        load(p_begin + PR_TILE, next);
        __syncthreads();
        int buf = 0;
        const int o = 32 * part_of; // this wave's 32 positions of a step
        for (int p0 = p_begin; p0 < p_end; p0 += PR_TILE) {
            const Pages after = pages_of(p0 + 2 * PR_TILE);
            const RowsLds<LO> &l = lds.step[buf];
            const int p = p0 + o, pa = part_of ? cur.of(2) : cur.of(0),
                      pb = part_of ? cur.of(3) : cur.of(1);
            if (partial(p0 + PR_TILE, next)) odd |= clean(p0 + PR_TILE, next);
            // (sx: the products with low parts, where those are scaled)
            f32x16 sv, sx;
#pragma unroll
            for (int e = 0; e < 16; ++e) sv[e] = sx[e] = 0.f;
            // Scores, with the next step's rows converted between their products (the
            // matrix unit takes 32 cycles for each). Operands are read one product
            // ahead, and no further, by barriers to the compiler's scheduling: 512
            // tokens over 32012 positions take 394 us with them and 397 without in f32
            // pages, 250 either way in f16 ones.
            half8 ahi[2], alo[2];
            auto keys = [&](int kk) {
                ahi[kk & 1] = *reinterpret_cast<const half8 *>(&l.khi[o + c][16 * kk + 8 * h]);
                if constexpr (LO)
                    alo[kk & 1] = *reinterpret_cast<const half8 *>(&l.klo[o + c][16 * kk + 8 * h]);
            };
            keys(0);
#pragma unroll
            for (int kk = 0; kk < KV_D / 16; ++kk) {
                if (kk + 1 < KV_D / 16) keys(kk + 1);
                if constexpr (LO) {
                    sx = mfma(ahi[kk & 1], qlo[kk], sx);
                    sv = mfma(ahi[kk & 1], qhi[kk], sv);
                    sx = mfma(alo[kk & 1], qhi[kk], sx);
                } else {
                    sv = mfma(ahi[kk & 1], qhi[kk], sv);
                    sv = mfma(ahi[kk & 1], qlo[kk], sv);
                }
                if (kk < 2 * R::N) store(buf ^ 1, kk);
                __builtin_amdgcn_sched_barrier(0);
            }
            load(p0 + 2 * PR_TILE, after);
            if constexpr (LO) sv += sx * (1.f / LO_SCALE);
            if (p + 31 > wave_all || (pa | pb) < 0) { // mask
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int pos = p + 8 * (e >> 2) + 4 * h + (e & 3);
                    sv[e] = pos <= sees && (e < 8 ? pa : pb) >= 0 ? sv[e] : -INFINITY;
                }
            }
            float tmax = sv[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) tmax = fmaxf(tmax, sv[e]);
            // The running maximum follows only when a score passes it by 2^8 or
            // more: until then weights are at most 2^8 times the first, and the 64
            // products that bring the sums to a new one are rare (in 32 rows of
            // equal chances some row has a new maximum in most steps). m_run lies 7
            // below the maximum, so that weights go up to 2^15: their f16 parts
            // resolve 2^-25, which is 2^-32 of the first weight. (Many equal small
            // weights are rounded the same way, and their errors add up.)
            const float m_new = fmaf(wave::max_halves(tmax), qscale, -7.f);
            if (__any(m_new > m_run + 8.f)) {
                const float m = fmaxf(m_run, m_new);
                const float corr = m == m_run ? 1.f : __builtin_amdgcn_exp2f(m_run - m);
#pragma unroll
                for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[j][e] *= corr;
                l_run *= corr;
                m_run = m;
            }
            const float base = m_run == -INFINITY ? 0.f : m_run; // (nothing seen yet: zero weights)
            float rs[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sv[e] = __builtin_amdgcn_exp2f(fmaf(sv[e], qscale, -base));
                rs[e & 1] += sv[e];
            }
            l_run += rs[0] + rs[1];
            // operand element 4 x + i of product (kk, j): position 16 kk + 8 x + 4 h + i,
            // which is the lane's weight 8 kk + 4 x + i
            half8 vhi[4], vlo[4];
            auto values = [&](int n) {
                const int kk = n >> 2, j = n & 3;
                const int vr = o + 16 * kk + 4 * h + ((lane & 15) >> 2);
                const int vd = 32 * j + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                const half4 x = read_transposed(&l.vhi[vr][vd]),
                            y = read_transposed(&l.vhi[vr + 8][vd]);
                vhi[n & 3] = half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                if constexpr (LO) {
                    const half4 z = read_transposed(&l.vlo[vr][vd]),
                                w = read_transposed(&l.vlo[vr + 8][vd]);
                    vlo[n & 3] = half8{z[0], z[1], z[2], z[3], w[0], w[1], w[2], w[3]};
                }
            };
            half8 phi, plo, pls; // (pls: the weights of the values' low parts)
            values(0);
            values(1);
#pragma unroll
            for (int n = 0; n < 8; n += 2) { // two products' sums in turn
                if ((n & 3) == 0) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        half2 hi, lo;
                        split2(sv[2 * n + i], sv[2 * n + i + 1], hi, lo);
                        phi[i] = hi[0];
                        phi[i + 1] = hi[1];
                        plo[i] = lo[0];
                        plo[i + 1] = lo[1];
                    }
                    if constexpr (LO) pls = phi * (_Float16)(1.f / LO_SCALE);
                }
                if (n + 2 < 8) {
                    values(n + 2);
                    values(n + 3);
                }
                f32x16 &d = acc[n & 3], &e = acc[(n + 1) & 3];
                d = mfma(vhi[n & 3], phi, d);
                e = mfma(vhi[(n + 1) & 3], phi, e);
                d = mfma(vhi[n & 3], plo, d);
                e = mfma(vhi[(n + 1) & 3], plo, e);
                if constexpr (LO) {
                    d = mfma(vlo[n & 3], pls, d);
                    e = mfma(vlo[(n + 1) & 3], pls, e);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __syncthreads();
            cur = next;
            next = after;
            buf ^= 1;
        }
        if (__syncthreads_or(odd)) {
            // the values left out, for the rows that see them: whatever its weight,
            // such a value makes the sum not finite (as it does in a step that all
            // rows see whole)
            for (int p0 = p_begin; p0 < p_end; p0 += PR_TILE) {
                const Pages pg = pages_of(p0);
                if (!partial(p0, pg)) continue;
                for (int i = 0; i < 32; ++i) {
                    const int pos = p0 + 32 * part_of + i;
                    const int e = i < 16 ? (part_of ? pg.of(2) : pg.of(0))
                                         : (part_of ? pg.of(3) : pg.of(1));
                    if (pos > sees || e < 0) continue;
                    const T *vb = (const T *)kv.pages + (size_t)e * psize +
                                  (size_t)(kv.kvh + kh) * hsize + (size_t)(pos & pmask) * KV_D;
#pragma unroll
                    for (int j = 0; j < KV_D / 32; ++j) {
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            const float v = (float)vb[32 * j + 8 * (x >> 2) + 4 * h + (x & 3)];
                            acc[j][x] += has_parts(v) ? 0.f : v * INFINITY;
                        }
                        asm volatile("" ::: "memory"); // (few loads at once: a rare path)
                    }
                }
            }
        }

        // the two halves' rows joined, in the first half's waves
        l_run = wave::sum_halves(l_run);
        if (part_of) {
            float(*o)[64] = lds.join[rows];
            o[0][lane] = m_run;
            o[1][lane] = l_run;
#pragma unroll
            for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[2 + 16 * j + e][lane] = acc[j][e];
        }
        __syncthreads();
        if (part_of || !ok) continue;
        {
            const float(*o)[64] = lds.join[rows];
            const float m2 = o[0][lane], m = fmaxf(m_run, m2), base = m == -INFINITY ? 0.f : m;
            const float a = __builtin_amdgcn_exp2f(m_run - base),
                        b = __builtin_amdgcn_exp2f(m2 - base);
            l_run = l_run * a + o[1][lane] * b;
            m_run = m;
#pragma unroll
            for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    acc[j][e] = acc[j][e] * a + o[2 + 16 * j + e][lane] * b;
        }
        float *dst = out + row * KV_D;
        float f = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f; // (saw nothing: zeros)
        if (piece.part >= 0) {
            dst = rs.parts + (((size_t)piece.part * kv.kvh + kh) * PR_ROWS + r) * PAGED_PART;
            if (h == 0) {
                dst[0] = m_run;
                dst[1] = l_run;
            }
            dst += 4;
            f = 1.f;
        }
#pragma unroll
        for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4 *>(dst + 32 * j + 8 * g + 4 * h) =
                    make_float4(acc[j][4 * g] * f, acc[j][4 * g + 1] * f, acc[j][4 * g + 2] * f,
                                acc[j][4 * g + 3] * f);
    }
}

} // namespace

int launch_paged_rows(const PagedKv &kv, const RowsScratch &rs, const float *q, float *out,
                      void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(max_pieces(rs.cap, kv.kvh) * kv.kvh); // (more groups there are not)
    const bool whole = 1 << kv.shift >= PR_TILE;
    auto kernel = whole ? paged_rows_kernel<float, true> : paged_rows_kernel<float, false>;
    if (kv.f16)
        kernel = whole ? paged_rows_kernel<_Float16, true> : paged_rows_kernel<_Float16, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(PR_THREADS), 0, st, kv, rs, q, out);
    return (int)hipGetLastError();
}

} // namespace hyq
