// Attention over 8-bit pages for slots of few new rows: the stream of
// hyq_paged_few.hip over codes and scales.
//
//   o_r = sum_t p_rt b_t v_t / sum_t p_rt,   p_rt = 2^(s_rt - m_r),
//   s_rt = log2(e) / sqrt(128) a_t q_r . k_t,
//
// with the codes k_t, v_t and the scales a_t, b_t of position t. Both products
// take the codes exactly:
//
// Scores on v_mfma_i32_16x16x64_i8, the keys' codes as they lie in memory. A
// row of queries is rounded to 22 bits below its power of two, q = 2^(e - 21) Q,
// and Q split into three signed bytes, whose products with the codes are whole
// numbers: three products of 64 dims each, nothing is converted, and sums of
// codes are exact. Then S^T [16 pos x 16 rows] is scaled by a_t.
//
// Sums on v_mfma_f32_16x16x32_f16, O^T [16 dims x 16 rows] += V^T . (p b)^T over
// 32 positions. A lane's weights are its operand as they are, its positions
// 16 t + 4 g + e the operand's places 8 g + 4 t + e. The values' operand wants
// eight positions of a dim in a lane: a lane loads eight dims of each of its
// positions, and one byte permutation per pair of positions picks a dim's two
// codes into the low bytes of two halves, u 2^-24 as f16, which an fma makes
// (u - 128) 2^-9. The weights' two f16 parts keep 22 bits: p lies up to 2^14 over
// the power of two that passes all scales the row has seen, and p b below 2^14, so
// that its error is at most 2^-39 of the largest. (Where the scales pass 2^32, p lies
// over 2^32 and b is brought down by the rest: an exponential below f32's normal
// numbers is zero, and so none above 2^-108 of the largest is.)
//
// Bound by memory, 264 bytes a position and head, and for few positions by loads that
// wait for each other and the merge's launch. With the merge: 64 slots of up to 8192
// positions, 32 heads over 8, 85 us for 438 MB (5.2 TB/s; this launch 81, VALU work 34
// and MFMAs 11 % of it); four of up to 60001, 16 over 4, 44 us for 165 MB (this launch
// 37); two of up to 1100, 10.7 us, of which the merge 4.6.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "hyq_paged_attn.hpp"
#include "hyq_wave.hpp"

namespace hyq {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int TILE = 32; // positions of a step, two of 16 (a page may end between them)
constexpr float LIFT = 14.f; // weights go up to 2^LIFT

// A row's queries as 22-bit whole numbers in three signed bytes, lowest first;
// lane (c, g): row c, dims 64 j + 16 g + b (so that a load of keys takes 64 bytes of
// a row from four lanes).
struct Query {
    i32x4 digit[3][2];
    float scale; // of the numbers, with log2(e) / sqrt(128); NaN for a row that is not finite
    __device__ __forceinline__ void form(const f32x4 (&v)[8], bool ok)
    {
        float x[32];
        float mx = 0.f; // (a NaN stays one)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                x[4 * i + b] = v[i][b];
                mx = wave::nmax(mx, fabsf(v[i][b]));
            }
        int lo, hi;
        wave::swap32(__builtin_bit_cast(int, wave::nmax_rows2(mx)), lo, hi);
        mx = wave::nmax(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
        const int e = query_exponent(mx);
        scale = ldexpf(1.4426950408889634f * 0.08838834764831845f, e - 21);
        if (!(mx < INFINITY)) scale = __builtin_nanf("");
        const float up = ok ? ldexpf(1.f, 21 - e) : 0.f;
        // A number is rounded by adding 1.5 * 2^23, whose last bit is 1, and with 128
        // added to each of its bytes these are the digits but for their upper bits.
        constexpr unsigned SIGNS = 0x808080u, ONE = 0x4b400000u; // (1.5 * 2^23)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                unsigned n[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const float y = fminf(x[16 * j + 4 * w + b] * up, 4194303.f) + 12582912.f;
                    n[b] = (__builtin_bit_cast(unsigned, y) + (SIGNS - ONE)) ^ SIGNS;
                }
                // the four numbers' bytes 0 and 1, and 2, by pairs; then by fours
                const unsigned a = __builtin_amdgcn_perm(n[1], n[0], 0x05010400u),
                               b = __builtin_amdgcn_perm(n[3], n[2], 0x05010400u),
                               c = __builtin_amdgcn_perm(n[1], n[0], 0x0c0c0602u),
                               d = __builtin_amdgcn_perm(n[3], n[2], 0x06020c0cu);
                digit[0][j][w] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
                digit[1][j][w] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
                digit[2][j][w] = (int)(c | d);
            }
    }
};

// A step's codes and scales of one KV head.
struct Step {
    i32x4 k[2][2]; // position 16 t + lane % 16, dims 64 j + 16 g ..
    u32x2 v[8];    // position 16 t + 4 g + e (4 t + e), dims 8 (lane % 16) ..
    f32x4 a[2], b[2]; // the scales of positions 16 t + 4 g ..
};

__device__ __forceinline__ i32x4 product(const i32x4 &k, const i32x4 &q, const i32x4 &c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q, c, 0, 0, 0);
}

// (u - 128) 2^-9 of byte x of two positions' words: u 2^-24 is u as the bits of
// an f16, subnormal, and the fma is exact.
__device__ __forceinline__ half2 values(unsigned first, unsigned second, int x)
{
    const unsigned pick = 0x0c000c00u | (unsigned)(4 + x) << 16 | (unsigned)x;
    const half2 h = __builtin_bit_cast(half2, __builtin_amdgcn_perm(second, first, pick));
    return __builtin_elementwise_fma(h, half2{(_Float16)32768.f, (_Float16)32768.f},
                                     half2{(_Float16)-0.25f, (_Float16)-0.25f});
}

template <bool SHARED>
__global__ __launch_bounds__(64 * FEW_WAVES, SHARED ? 3 : 2) void paged_few_q8_kernel(
    PagedKv kv, int few_rows, int max_workers, RowsScratch rs, SharedPlan sp,
    const float *__restrict__ q, int part_rows, float *__restrict__ part,
    int2 *__restrict__ shared, float *__restrict__ out)
{
    extern __shared__ long long before[]; // [seqs + 1]
    __shared__ long long wsum[4];
    if (blockIdx.x * FEW_WAVES >= max_workers) { // one more workgroup: the tile form's plan
        rows_plan(kv, few_rows, rs, (int *)before);
        return;
    }
    FewPlan plan;
    if constexpr (!SHARED) plan = few_plan<TILE>(kv, few_rows, max_workers, before, wsum);
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    int workers, w;
    if constexpr (SHARED) { // whole workgroups, and the last waves alike on a CU's SIMDs
        workers = min(sp.head->workers, sp.few_most);
        const int groups = (workers + 256 * FEW_WAVES - 1) / (256 * FEW_WAVES) * 256;
        w = (int)blockIdx.x < groups
                ? blockIdx.x + groups * (((threadIdx.x >> 6) + (blockIdx.x >> 8)) & 3)
                : workers;
    } else {
        workers = plan.workers;
        w = blockIdx.x + max_workers / FEW_WAVES * (threadIdx.x >> 6);
    }
    w = __builtin_amdgcn_readfirstlane(w);
    if (w >= workers) return;
    long long at = SHARED ? 0 : plan.begin(w);
    const long long stop = SHARED ? 1 : plan.begin(w + 1);
    const int rep = kv.heads / kv.kvh;
    const size_t hsize = (size_t)KV_D << kv.shift; // a head's codes of a page
    const size_t psize = 2 * kv.kvh * (hsize / KV_D * kv_row_bytes(KV_T_Q8));
    const int pmask = (1 << kv.shift) - 1;

    int s = 0; // the slot that holds tile `at`: the last with before[s] <= at
    if constexpr (!SHARED) {
        int hi = kv.seqs;
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (before[mid] <= at) s = mid;
            else hi = mid;
        }
    }
    while (at < stop) {
        SlotRows sr;
        int kh, t0, t1, tiles = 0, skip = 0;
        bool narrow = false; // a block of several slots' rows, which see all positions
        bool whole; // no other worker's part, and no prefix's, is to be joined
        if constexpr (SHARED) {
            const FewPiece f = few_piece<TILE>(kv, sp, w);
            if (!f.narrow && f.n > few_rows) return;
            s = f.slot, kh = f.kh, t0 = f.t0, t1 = f.t1, skip = f.skip;
            sr = SlotRows{f.begin, f.n, f.len};
            whole = f.ways == 1 && skip == 0 && !f.narrow;
            narrow = f.narrow != 0;
            at = stop;
        } else {
            while (before[s + 1] <= at) ++s; // slots without tiles
            s = __builtin_amdgcn_readfirstlane(s);
            sr = slot_rows(kv, s);
            tiles = slot_tiles<TILE>(sr.len);
            const int in = __builtin_amdgcn_readfirstlane((int)(at - before[s]));
            kh = in / tiles, t0 = in % tiles;
            t1 = __builtin_amdgcn_readfirstlane((int)min((long long)tiles, t0 + (stop - at)));
            whole = t0 == 0 && t1 == tiles;
            at += t1 - t0;
        }

        // this lane's row: token c / rep of the slot's new rows
        const int tok = c / rep;
        bool ok = tok < sr.n;
        const int head = kh * rep + c % rep;
        int packed = sr.begin + (ok ? tok : 0);
        int sees = ok ? sr.len - sr.n + tok : -1; // this row's last visible position
        if constexpr (SHARED) {
            if (narrow) {
                const int listed = ok ? sp.list[packed] : -1;
                ok = (unsigned)listed < (unsigned)kv.rows;
                packed = ok ? listed : 0;
                sees = ok ? sr.len - 1 : -1;
            }
        }
        const size_t row = (size_t)packed * kv.heads + head;
        f32x4 qrow[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            qrow[i] = *reinterpret_cast<const f32x4 *>(q + row * KV_D + 64 * (i >> 2) + 16 * g +
                                                       4 * (i & 3));
        Query query;
        query.form(qrow, ok);
        f32x4 acc[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        // m: the running maximum less LIFT; top: a power of two above all scales of
        // values seen (not below 2^-88, that sums of weights over it be numbers);
        // log_top: its logarithm as it enters the weights (not above Q8_LOG_MOST)
        float m = -INFINITY, l = 0.f, top = 0x1p-88f, log_top = -88.f;

        const int *entries = kv.table + (size_t)s * kv.stride;
        int have = -64, ids = -1; // lane i: the slot's page have + i
        auto page_of = [&](int p0) { // the page of 16 positions, -1 where there is none
            const int p = p0 >> kv.shift;
            if (p - have >= 64 || p < have) {
                have = p;
                ids = have + lane < kv.stride ? entries[have + lane] : -1;
            }
            const int id = __builtin_amdgcn_readlane(ids, p - have);
            return p0 < sr.len && (unsigned)id < (unsigned)kv.npages ? id : -1;
        };
        struct Pages {
            int id[2];
        };
        auto pages_of = [&](int p0) {
            Pages p;
            p.id[0] = page_of(p0);
            p.id[1] = page_of(p0 + 16);
            return p;
        };
        auto base_of = [&](int page) {
            return (const unsigned char *)kv.pages + (size_t)max(page, 0) * psize;
        };
        // (Loads are unconditional: behind the length they read what the page holds
        // there, and without a page the pool's first; codes are always numbers, and
        // scales count where the row sees the position.)
        Step st;
        auto load_k = [&](auto once, int p0, const Pages &pg) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const unsigned char *b = base_of(pg.id[t]);
                const int p = (p0 + 16 * t) & pmask;
                const unsigned char *kb = b + kh * hsize;
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    st.k[t][j] = cached<i32x4, once.value>(kb, (p + c) * KV_D + 64 * j + 16 * g);
                st.a[t] = cached<f32x4, once.value>(
                    (const float *)(b + 2 * kv.kvh * hsize) + ((size_t)kh << kv.shift), p + 4 * g);
            }
        };
        auto load_v = [&](auto once, int p0, const Pages &pg) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const unsigned char *b = base_of(pg.id[t]);
                const int p = (p0 + 16 * t) & pmask;
                const unsigned char *vb = b + (kv.kvh + kh) * hsize;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    st.v[4 * t + e] =
                        cached<u32x2, once.value>(vb, (p + 4 * g + e) * KV_D + 8 * c);
                st.b[t] = cached<f32x4, once.value>((const float *)(b + 2 * kv.kvh * hsize) +
                                                        ((size_t)(kv.kvh + kh) << kv.shift),
                                                    p + 4 * g);
            }
        };
        const int p_begin = skip + t0 * TILE;
        // (pages that a neighbouring slot names too are kept in the caches)
        const int at0 = min(p_begin >> kv.shift, kv.stride - 1);
        const int mine = entries[at0], below = s ? entries[at0 - kv.stride] : -1,
                  above = s + 1 < kv.seqs ? entries[at0 + kv.stride] : -1;
        Pages pages = pages_of(p_begin);
        const bool alone =
            __builtin_amdgcn_readfirstlane(mine != below && mine != above && !narrow) != 0;
        auto stream = [&](auto once) {
            load_k(once, p_begin, pages);
            load_v(once, p_begin, pages);
            for (int t = t0; t < t1; ++t) {
                const int p0 = skip + t * TILE, pn = skip + min(t + 1, t1 - 1) * TILE;
                float sv[8], b[8];
                float mx = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    i32x4 n[3] = {};
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 3; ++i)
                            n[i] = product(st.k[h][j], query.digit[i][j], n[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // (each sum is below 2^21, a number of f32)
                        const float dot = fmaf((float)n[2][e], 65536.f,
                                               fmaf((float)n[1][e], 256.f, (float)n[0][e]));
                        const bool see = p0 + 16 * h + 4 * g + e <= sees && pages.id[h] >= 0;
                        const float x = dot * (st.a[h][e] * query.scale);
                        sv[4 * h + e] = see ? x : -INFINITY;
                        b[4 * h + e] = see ? st.b[h][e] : 0.f;
                        mx = fmaxf(mx, sv[4 * h + e]);
                    }
                }
                const Pages next = pages_of(pn);
                load_k(once, pn, next);
                float bm = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) bm = fmaxf(bm, b[i]);
                mx = wave::max_halves(wave::max_rows2(mx));
                bm = wave::max_halves(wave::max_rows2(bm));
                const float mn = fmaxf(m, mx - LIFT);
                if (__any(mn != m || bm > top)) {
                    const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                    const Q8Top to = q8_top(bm, top, log_top);
                    l = l * corr * to.weights; // (in turn: their product may be too small)
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[x] *= corr * to.sums;
                    m = mn;
                }
                if (__any(top > Q8_MOST)) { // (rare)
                    const float rest = q8_rest(top);
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[i] *= rest;
                }
                // a row that has seen nothing yet keeps zero weights
                const float base = m == -INFINITY ? 0.f : m + log_top;
                half8 hi, lo;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(sv[i] - base),
                                p1 = __builtin_amdgcn_exp2f(sv[i + 1] - base);
                    sum += p0 + p1;
                    half2 x, y;
                    split2(p0 * b[i], p1 * b[i + 1], x, y);
                    hi[i] = x[0];
                    hi[i + 1] = x[1];
                    lo[i] = y[0];
                    lo[i + 1] = y[1];
                }
                l += sum;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    half8 vt;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const half2 y = values(st.v[i][x >> 2], st.v[i + 1][x >> 2], x & 3);
                        vt[i] = y[0];
                        vt[i + 1] = y[1];
                    }
                    acc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, hi, acc[x], 0, 0, 0);
                    acc[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, lo, acc[x], 0, 0, 0);
                }
                load_v(once, pn, next);
                pages = next;
            }
        };
        if (alone) stream(std::true_type{});
        else stream(std::false_type{});
        l = wave::sum_halves(wave::sum_rows2(l));
        if (!SHARED && t0 == 0 && lane == 0) { // who shares the unit, for the merge
            const long long last = before[s] + (long long)(kh + 1) * tiles - 1;
            const int n = t1 == tiles ? 1 : plan.worker(last) - w + 1;
            shared[(size_t)s * kv.kvh + kh] = make_int2(w, n);
        }
        float *o, f;
        if (whole) {
            // (a row that saw nothing gives zeros)
            o = out + row * KV_D;
            f = l > 0.f || l != l ? 512.f / (l * q8_rest(top)) : 0.f;
        } else {
            const long long slot = SHARED ? w : (long long)w + (long long)s * kv.kvh + kh;
            o = part + ((size_t)slot * part_rows + c) * PAGED_PART;
            if (ok && g == 0) { // (weights of at most 2^-24, see Q8_DOWN)
                o[0] = m + (LIFT + Q8_DOWN);
                o[1] = l * (fminf(top, Q8_MOST) * 0x1p-38f);
            }
            o += 4;
            f = top * 0x1p-29f;
        }
        if (ok) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float4 *>(o + 32 * g + 8 * e + 4 * h) =
                        make_float4(acc[4 * h][e] * f, acc[4 * h + 1][e] * f,
                                    acc[4 * h + 2][e] * f, acc[4 * h + 3][e] * f);
        }
    }
}

} // namespace

int launch_paged_few_q8(const PagedKv &kv, int few, int workers, const RowsScratch &rs,
                        const SharedPlan *sp, const float *q, int part_rows, float *part,
                        int2 *shared, float *out, void *stream)
{
    const size_t lds = ((size_t)kv.seqs + 1) * 8;
    const dim3 grid(workers / FEW_WAVES + (rs.cap > 0)), block(64 * FEW_WAVES);
    auto kernel = sp ? paged_few_q8_kernel<true> : paged_few_q8_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, block, lds, (hipStream_t)stream, kv, few, workers, rs,
                       sp ? *sp : SharedPlan{}, q, part_rows, part, shared, out);
    return (int)hipGetLastError();
}

} // namespace hyq
