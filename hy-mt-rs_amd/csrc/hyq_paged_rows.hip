// Attention over a paged cache for slots of many new rows (prompts): causal,
// on the matrix cores, for a ragged batch.
//
// A workgroup takes the query rows of one KV head for a block of a slot's new
// tokens - 128 rows, row r = token r / rep of the block, query head r % rep of
// the group - and a range of 32-position tiles. Each of its four waves owns 32
// rows and forms transposed products with v_mfma_f32_32x32x16_f16, so that a
// lane holds one query row (lane % 32) and 16 of its positions or dims:
//   S^T [32 pos x 32 rows]   = K_tile . Q^T
//   O^T [128 dims x 32 rows] += V_tile^T . P^T
// with the softmax's running maximum and sum per lane (one exchange between
// the row's two lanes). An f32 operand x is split into f16 parts hi = f16(x),
// lo = f16(x - hi) and products sum hi.hi + lo.hi + hi.lo in f32, which keeps
// the scores and sums near f32 accuracy; f16 pages are exact as they are and
// need no low parts of keys and values. f32 pages hold values below 65504.
//
// Blocks of different slots and places see very different numbers of tiles, so
// a plan cuts them: one workgroup counts every block's tiles and makes pieces
// of about equal length, enough to fill the GPU, and the pieces of a block
// that was cut leave partial rows, which a merge joins in order.
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

constexpr int PR_ROWS = 128;        // query rows per workgroup
constexpr int PR_TILE = 32;         // positions per tile
constexpr int PR_KP = KV_D + 8;     // K tile row pitch (halves)
constexpr int PR_VP = PR_TILE + 8;  // V^T tile row pitch (halves)
constexpr int PR_FILL = 512;        // workgroups that fill the GPU: two per CU
constexpr int PR_MIN_TILES = 4;     // the shortest piece worth its partial rows

// The plan in scratch: counts, the blocks, then the pieces.
struct Block {
    int slot, index, part, pieces; // first partial block and pieces of the block
};
struct Piece {
    int block, t0, t1, part; // part: the partial block it writes, -1 for the output
};
struct Plan {
    int blocks, pieces, parts, unused;
};

int max_blocks(int seqs, int rows, int tq) { return rows / tq + std::min(seqs, rows); }
// sum of ceil(n / each) with each >= kvh tiles / PR_FILL; a block that is cut
// (n > each) has fewer than 2 n / each pieces
int max_pieces(int blocks, int kvh) { return blocks + PR_FILL / kvh + 1; }
int max_parts(int kvh) { return 2 * (PR_FILL / kvh + 1); }

__device__ __forceinline__ int block_tiles(const SlotRows &r, int b, int tq)
{
    const int last = r.len - r.n + min(r.n, (b + 1) * tq); // one past the last position seen
    return max(1, (last + PR_TILE - 1) / PR_TILE);
}

// Exclusive scan of one value per thread over 1024 threads; returns the total.
__device__ __forceinline__ int scan1024(int mine, int &before, int *wsum)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int v = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        if (w < wave) base += wsum[w];
        all += wsum[w];
    }
    before = base + v - mine;
    return all;
}

// One workgroup of 1024 threads. Dynamic LDS: seqs ints.
__global__ __launch_bounds__(1024) void paged_rows_plan_kernel(PagedKv kv, int few_rows, int tq,
                                                               int cap, Plan *plan,
                                                               Block *blocks, Piece *pieces)
{
    extern __shared__ int first[]; // a slot's first block
    __shared__ int wsum[16];
    const int t = threadIdx.x;
    int count = 0;
    for (int b = 0; b < kv.seqs; b += 1024) {
        int nb = 0, before;
        if (b + t < kv.seqs) {
            const SlotRows r = slot_rows(kv, b + t);
            nb = r.n > few_rows ? (r.n + tq - 1) / tq : 0;
        }
        const int all = scan1024(nb, before, wsum);
        if (b + t < kv.seqs) first[b + t] = count + before;
        count += all;
    }
    // (starts that do not ascend could claim rows twice: what the scratch has
    // no room for is left out)
    count = min(count, cap);
    __syncthreads();
    auto slot_of = [&](int u) {
        int s = 0, hi = kv.seqs; // the last slot with first[s] <= u
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (first[mid] <= u) s = mid;
            else hi = mid;
        }
        return s;
    };
    // all tiles of one KV head (a block has at most 2^24 / 32, so that 1024 of
    // them fit an int)
    long long tiles = 0;
    for (int b = 0; b < count; b += 1024) {
        int mine = 0, before;
        if (b + t < count) {
            const int s = slot_of(b + t);
            mine = block_tiles(slot_rows(kv, s), b + t - first[s], tq);
        }
        tiles += scan1024(mine, before, wsum);
    }
    const int each = max((long long)PR_MIN_TILES, (tiles * kv.kvh + PR_FILL - 1) / PR_FILL);
    int npieces = 0, nparts = 0;
    for (int b = 0; b < count; b += 1024) {
        int s = 0, n = 0, k = 0, before, pbefore;
        if (b + t < count) {
            s = slot_of(b + t);
            n = block_tiles(slot_rows(kv, s), b + t - first[s], tq);
            k = (n + each - 1) / each;
        }
        const int all = scan1024(k, before, wsum);
        const int pall = scan1024(k > 1 ? k : 0, pbefore, wsum);
        if (b + t < count) {
            blocks[b + t] = Block{s, b + t - first[s], nparts + pbefore, k};
            for (int i = 0; i < k; ++i)
                pieces[npieces + before + i] =
                    Piece{b + t, (int)((long long)n * i / k), (int)((long long)n * (i + 1) / k),
                          k > 1 ? nparts + pbefore + i : -1};
        }
        npieces += all;
        nparts += pall;
    }
    if (t == 0) *plan = Plan{count, npieces, nparts, 0};
}

__device__ __forceinline__ f32x16 mfma(const half8 &a, const half8 &b, const f32x16 &c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void split_f16(float x, _Float16 &hi, _Float16 &lo)
{
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}
__device__ __forceinline__ int fbits(float v) { return __builtin_bit_cast(int, v); }
__device__ __forceinline__ float bitsf(int v) { return __builtin_bit_cast(float, v); }

template <class T> struct Four;
template <> struct Four<float> {
    typedef float4 type;
    static __device__ __forceinline__ void get(const float4 &v, float (&x)[4])
    {
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    }
};
template <> struct Four<_Float16> {
    typedef half4 type;
    static __device__ __forceinline__ void get(const half4 &v, float (&x)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
    }
};

template <class T>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(
    PagedKv kv, int tq, const Plan *__restrict__ plan, const Block *__restrict__ blocks,
    const Piece *__restrict__ pieces, const float *__restrict__ q, float *__restrict__ part,
    float *__restrict__ out)
{
    constexpr bool LO = sizeof(T) == 4; // low parts of keys and values
    typedef typename Four<T>::type Vec;
    __shared__ __align__(16) _Float16 Khi[PR_TILE][PR_KP];
    __shared__ __align__(16) _Float16 Klo[LO ? PR_TILE : 1][PR_KP];
    __shared__ __align__(16) _Float16 Vhi[KV_D][PR_VP];
    __shared__ __align__(16) _Float16 Vlo[LO ? KV_D : 1][PR_VP];
    if ((int)blockIdx.y >= plan->pieces) return;
    const Piece piece = pieces[blockIdx.y];
    const Block blk = blocks[piece.block];
    const int kh = blockIdx.x, s = blk.slot;
    const SlotRows sr = slot_rows(kv, s);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, h = lane >> 5;
    const int rep = kv.heads / kv.kvh;
    const size_t hsize = (size_t)KV_D << kv.shift, psize = 2 * hsize * kv.kvh;
    const int pmask = (1 << kv.shift) - 1;
    const float sc = 1.4426950408889634f * 0.08838834764831845f;

    const int tok0 = blk.index * tq;
    const int first = sr.len - sr.n;            // position of the slot's first new row
    const int toks = min(tq, sr.n - tok0);
    const int p_end = min(piece.t1 * PR_TILE, first + tok0 + toks);

    // this lane's query row
    const int r = 32 * wave + (lane & 31);
    const int tl = r / rep;
    const bool ok = tl < toks;
    const int head = kh * rep + r % rep;
    const int sees = ok ? first + tok0 + tl : -1; // its last visible position
    // the wave's last visible position, and the block's first row's
    const int wave_last = first + tok0 + min(toks - 1, (32 * wave + 31) / rep);
    const int all_see = first + tok0;
    const size_t row = (size_t)(sr.begin + tok0 + (ok ? tl : 0)) * kv.heads + head;

    // q = 2^e (hi + lo), the row's power of two bringing it inside f16's range
    half8 qhi[KV_D / 16], qlo[KV_D / 16];
    float qscale;
    {
        const float *qr = q + row * KV_D + 8 * h;
        float mx = 0.f;
        for (int kk = 0; kk < KV_D / 16; ++kk)
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(qr[16 * kk + i]));
        mx = wave::max_halves(mx);
        const int e = mx > 0.f && mx < INFINITY ? ilogbf(mx) : 0;
        qscale = ldexpf(sc, e);
        const float inv = ldexpf(1.f, -e);
#pragma unroll
        for (int kk = 0; kk < KV_D / 16; ++kk)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = ok ? qr[16 * kk + i] * inv : 0.f;
                _Float16 hi, lo;
                split_f16(y, hi, lo);
                qhi[kk][i] = hi;
                qlo[kk][i] = fabsf(y) < INFINITY ? lo : (_Float16)0.f;
            }
    }

    // tile loads: thread t fetches four dims (d4) of rows {2pp, 2pp+1, 2pp+16, 2pp+17}
    const int d4 = t & 31, pp = t >> 5;
    const int *entries = kv.table + (size_t)s * kv.stride;
    // the pages of a tile's two 16-position halves, -1 where none
    auto entry = [&](int p) {
        if (p >= p_end) return -1;
        const int e = entries[p >> kv.shift];
        return (unsigned)e < (unsigned)kv.npages ? e : -1;
    };
    Vec kr[4], vr[4];
    auto load_tile = [&](int p0, const int (&pg)[2]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = p0 + 2 * pp + (j & 1) + 16 * (j >> 1);
            const int e = pg[j >> 1];
            Vec z{};
            kr[j] = z;
            vr[j] = z;
            if (e >= 0 && p < p_end) {
                const T *b = (const T *)kv.pages + (size_t)e * psize + (size_t)kh * hsize +
                             (size_t)(p & pmask) * KV_D + 4 * d4;
                kr[j] = *reinterpret_cast<const Vec *>(b);
                vr[j] = *reinterpret_cast<const Vec *>(b + hsize * kv.kvh);
            }
        }
    };
    // (clean: values that are not finite stay out of the products)
    auto store_tile = [&](bool clean) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int rr = 2 * pp + (j & 1) + 16 * (j >> 1);
            float x[4];
            Four<T>::get(kr[j], x);
            half4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                _Float16 a, b;
                split_f16(x[i], a, b);
                hi[i] = a;
                lo[i] = b;
            }
            *reinterpret_cast<half4 *>(&Khi[rr][4 * d4]) = hi;
            if constexpr (LO) *reinterpret_cast<half4 *>(&Klo[rr][4 * d4]) = lo;
        }
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
            const int rr = 2 * pp + 16 * jp;
            float x[4], y[4];
            Four<T>::get(vr[2 * jp], x);
            Four<T>::get(vr[2 * jp + 1], y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (clean) {
                    x[i] = fabsf(x[i]) < INFINITY ? x[i] : 0.f;
                    y[i] = fabsf(y[i]) < INFINITY ? y[i] : 0.f;
                }
                half2 hi, lo;
                _Float16 a, b;
                split_f16(x[i], a, b);
                hi[0] = a;
                lo[0] = b;
                split_f16(y[i], a, b);
                hi[1] = a;
                lo[1] = b;
                *reinterpret_cast<half2 *>(&Vhi[4 * d4 + i][rr]) = hi;
                if constexpr (LO) *reinterpret_cast<half2 *>(&Vlo[4 * d4 + i][rr]) = lo;
            }
        }
    };
    auto odd = [&]() { // whether this thread's values are not all finite
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x[4];
            Four<T>::get(vr[j], x);
#pragma unroll
            for (int i = 0; i < 4; ++i) z = fmaf(x[i], 0.f, z);
        }
        return z != 0.f;
    };

    f32x16 acc[KV_D / 32];
#pragma unroll
    for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    const int p_begin = piece.t0 * PR_TILE;
    int pg[2] = {entry(p_begin), entry(p_begin + 16)};
    int nx[2] = {entry(p_begin + PR_TILE), entry(p_begin + PR_TILE + 16)};
    load_tile(p_begin, pg);
    for (int p0 = p_begin; p0 < p_end; p0 += PR_TILE) {
        // a tile that some row sees in part: a value there that is not finite
        // must not reach the rows that do not see it (0 * inf). The barrier:
        // the previous tile's readers are done.
        bool careful = false;
        if (p0 + PR_TILE - 1 > all_see) careful = __syncthreads_or(odd());
        else __syncthreads();
        store_tile(careful);
        const int cur[2] = {pg[0], pg[1]};
        pg[0] = nx[0], pg[1] = nx[1];
        if (p0 + PR_TILE < p_end) {
            load_tile(p0 + PR_TILE, pg);
            nx[0] = entry(p0 + 2 * PR_TILE);
            nx[1] = entry(p0 + 2 * PR_TILE + 16);
        }
        __syncthreads();
        if (p0 > wave_last) continue; // every row of this wave is before the tile

        f32x16 sv;
#pragma unroll
        for (int e = 0; e < 16; ++e) sv[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KV_D / 16; ++kk) {
            const half8 ahi = *reinterpret_cast<const half8 *>(&Khi[lane & 31][16 * kk + 8 * h]);
            sv = mfma(ahi, qhi[kk], sv);
            sv = mfma(ahi, qlo[kk], sv);
            if constexpr (LO) {
                const half8 alo =
                    *reinterpret_cast<const half8 *>(&Klo[lane & 31][16 * kk + 8 * h]);
                sv = mfma(alo, qhi[kk], sv);
            }
        }
        // scale, mask, softmax (one row per lane pair)
        float tmax = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int p = p0 + 8 * (e >> 2) + 4 * h + (e & 3);
            sv[e] = p <= sees && cur[e >> 3] >= 0 ? sv[e] * qscale : -INFINITY;
            tmax = fmaxf(tmax, sv[e]);
        }
        const float m_new = fmaxf(m_run, wave::max_halves(tmax));
        const float base = m_new == -INFINITY ? 0.f : m_new; // (nothing seen yet: zero weights)
        const float corr = __builtin_amdgcn_exp2f(m_run - base);
        float rs = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sv[e] = __builtin_amdgcn_exp2f(sv[e] - base);
            rs += sv[e];
        }
        if (__any(m_new != m_run)) {
#pragma unroll
            for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[j][e] *= corr;
            l_run *= corr;
        }
        l_run += rs;
        m_run = m_new;

        // P^T operands: positions 16kk + 8h + (0..7) of this lane's row,
        // half from the partner lane (lane ^ 32)
#pragma unroll
        for (int kk = 0; kk < PR_TILE / 16; ++kk) {
            half8 phi, plo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto sw = __builtin_amdgcn_permlane32_swap(fbits(sv[8 * kk + i]),
                                                                 fbits(sv[8 * kk + 4 + i]),
                                                                 false, false);
                _Float16 a, b;
                split_f16(bitsf(sw[0]), a, b);
                phi[i] = a;
                plo[i] = b;
                split_f16(bitsf(sw[1]), a, b);
                phi[4 + i] = a;
                plo[4 + i] = b;
            }
#pragma unroll
            for (int j = 0; j < KV_D / 32; ++j) {
                const int d = 32 * j + (lane & 31);
                const half8 vhi = *reinterpret_cast<const half8 *>(&Vhi[d][16 * kk + 8 * h]);
                acc[j] = mfma(vhi, phi, acc[j]);
                acc[j] = mfma(vhi, plo, acc[j]);
                if constexpr (LO) {
                    const half8 vlo = *reinterpret_cast<const half8 *>(&Vlo[d][16 * kk + 8 * h]);
                    acc[j] = mfma(vlo, phi, acc[j]);
                }
            }
        }
        if (careful) { // the values left out, for the rows that see them
            for (int i = 0; i < PR_TILE; ++i) {
                const int src = (lane & 31) + 32 * ((i >> 2) & 1);
                float w = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = __shfl(sv[e], src, 64);
                    if (e == 4 * (i >> 3) + (i & 3)) w = x;
                }
                const int p = p0 + i, pe = cur[i >> 4];
                if (p > sees || pe < 0) continue;
                const T *vb = (const T *)kv.pages + (size_t)pe * psize +
                              (size_t)(kv.kvh + kh) * hsize + (size_t)(p & pmask) * KV_D;
#pragma unroll
                for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float v = (float)vb[32 * j + 8 * (e >> 2) + 4 * h + (e & 3)];
                        if (!(fabsf(v) < INFINITY)) acc[j][e] = fmaf(w, v, acc[j][e]);
                    }
            }
        }
    }
    if (!ok) return;
    l_run = wave::sum_halves(l_run);
    float *o = out + row * KV_D;
    float f = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f; // (saw nothing: zeros)
    if (piece.part >= 0) {
        o = part + (((size_t)piece.part * kv.kvh + kh) * PR_ROWS + r) * PAGED_PART;
        if (h == 0) {
            o[0] = m_run;
            o[1] = l_run;
        }
        o += 4;
        f = 1.f;
    }
#pragma unroll
    for (int j = 0; j < KV_D / 32; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4 *>(o + 32 * j + 8 * g + 4 * h) =
                make_float4(acc[j][4 * g] * f, acc[j][4 * g + 1] * f, acc[j][4 * g + 2] * f,
                            acc[j][4 * g + 3] * f);
}

// Joins the pieces of a block that was cut, in order. Grid (kv heads, blocks,
// PR_ROWS / 8): 8 rows, a 32-lane half wave each.
__global__ __launch_bounds__(256) void paged_rows_merge_kernel(
    PagedKv kv, int tq, const Plan *__restrict__ plan, const Block *__restrict__ blocks,
    const float *__restrict__ part, float *__restrict__ out)
{
    if ((int)blockIdx.y >= plan->blocks) return;
    const Block blk = blocks[blockIdx.y];
    if (blk.pieces < 2) return;
    const SlotRows sr = slot_rows(kv, blk.slot);
    const int rep = kv.heads / kv.kvh, kh = blockIdx.x;
    const int r = blockIdx.z * 8 + (threadIdx.x >> 5), d = 4 * (threadIdx.x & 31);
    const int tl = r / rep;
    if (tl >= min(tq, sr.n - blk.index * tq)) return;
    const size_t step = (size_t)kv.kvh * PR_ROWS * PAGED_PART;
    const float *p = part + (((size_t)blk.part * kv.kvh + kh) * PR_ROWS + r) * PAGED_PART;
    float M = -INFINITY;
    for (int i = 0; i < blk.pieces; ++i) M = fmaxf(M, p[i * step]);
    const float base = M == -INFINITY ? 0.f : M;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll 4
    for (int i = 0; i < blk.pieces; ++i) {
        const float x = __builtin_amdgcn_exp2f(p[i * step] - base);
        const float4 v = *reinterpret_cast<const float4 *>(p + i * step + 4 + d);
        den = fmaf(x, p[i * step + 1], den);
        num.x = fmaf(x, v.x, num.x);
        num.y = fmaf(x, v.y, num.y);
        num.z = fmaf(x, v.z, num.z);
        num.w = fmaf(x, v.w, num.w);
    }
    const float f = den > 0.f || den != den ? 1.f / den : 0.f;
    const size_t row = (size_t)(sr.begin + blk.index * tq + tl) * kv.heads + kh * rep + r % rep;
    *reinterpret_cast<float4 *>(out + row * KV_D + d) =
        make_float4(num.x * f, num.y * f, num.z * f, num.w * f);
}

struct RowsScratch {
    size_t blocks, pieces, parts, bytes;
};
RowsScratch rows_layout(int seqs, int kvh, int heads, int rows)
{
    const int nb = max_blocks(seqs, rows, PR_ROWS / (heads / kvh));
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    RowsScratch r;
    r.blocks = up(sizeof(Plan));
    r.pieces = r.blocks + up(nb * sizeof(Block));
    r.parts = r.pieces + up(max_pieces(nb, kvh) * sizeof(Piece));
    r.bytes = r.parts + up((size_t)max_parts(kvh) * kvh * PR_ROWS * PAGED_PART * 4);
    return r;
}

} // namespace

size_t paged_rows_scratch(int seqs, int kvh, int heads, int rows)
{
    return rows_layout(seqs, kvh, heads, rows).bytes;
}

int launch_paged_rows(const PagedKv &kv, const float *q, void *scratch, float *out, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const int rep = kv.heads / kv.kvh, tq = PR_ROWS / rep;
    const int nb = max_blocks(kv.seqs, kv.rows, tq);
    const RowsScratch l = rows_layout(kv.seqs, kv.kvh, kv.heads, kv.rows);
    char *base = (char *)scratch;
    Plan *plan = (Plan *)base;
    Block *blocks = (Block *)(base + l.blocks);
    Piece *pieces = (Piece *)(base + l.pieces);
    float *part = (float *)(base + l.parts);
    hipLaunchKernelGGL(paged_rows_plan_kernel, dim3(1), dim3(1024), (size_t)kv.seqs * 4, st,
                       kv, paged_few_rows(rep), tq, nb, plan, blocks, pieces);
    const dim3 grid(kv.kvh, max_pieces(nb, kv.kvh));
    if (kv.f16)
        hipLaunchKernelGGL(paged_rows_kernel<_Float16>, grid, dim3(256), 0, st, kv, tq, plan,
                           blocks, pieces, q, part, out);
    else
        hipLaunchKernelGGL(paged_rows_kernel<float>, grid, dim3(256), 0, st, kv, tq, plan, blocks,
                           pieces, q, part, out);
    hipLaunchKernelGGL(paged_rows_merge_kernel, dim3(kv.kvh, nb, PR_ROWS / 8), dim3(256), 0, st,
                       kv, tq, plan, blocks, part, out);
    return (int)hipGetLastError();
}

} // namespace hyq
