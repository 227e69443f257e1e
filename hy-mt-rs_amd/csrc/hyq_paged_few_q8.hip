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
// (u - 128) 2^-9. The weights' two f16 parts keep 22 bits: p lies up to 2^14 and
// b below the power of two that passes all scales the row has seen, so that a
// weight's error is at most 2^-39 of the largest.
//
// Bound by memory: 264 bytes a position and head.
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
// lane (c, g): row c, dims 32 g + 16 j + b.
struct Query {
    i32x4 digit[3][2];
    float scale; // of the numbers, with log2(e) / sqrt(128); NaN for a row that is not finite
    __device__ __forceinline__ void load(const float *row, bool ok, int g)
    {
        float x[32];
        float mx = 0.f, odd = 0.f; // (a sum of x * 0: NaN if one is not finite)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 v = *reinterpret_cast<const float4 *>(row + 32 * g + 4 * i);
            const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float y = ok ? w[b] : 0.f;
                x[4 * i + b] = y;
                mx = fmaxf(mx, fabsf(y));
                odd = fmaf(y, 0.f, odd);
            }
        }
        mx = wave::max_halves(wave::max_rows2(mx));
        odd = wave::sum_halves(wave::sum_rows2(odd));
        const int e = query_exponent(mx);
        scale = ldexpf(1.4426950408889634f * 0.08838834764831845f, e - 21) + odd;
        const float up = ldexpf(1.f, 21 - e);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                unsigned d[3] = {0, 0, 0};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    int n = (int)rintf(x[16 * j + 4 * w + b] * up); // below 2^22 in magnitude
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        const int low = (int)(signed char)n;
                        d[i] |= (unsigned)(low & 255) << (8 * b);
                        n = (n - low) >> 8;
                    }
                }
#pragma unroll
                for (int i = 0; i < 3; ++i) digit[i][j][w] = (int)d[i];
            }
    }
};

// A step's codes and scales of one KV head.
struct Step {
    i32x4 k[2][2]; // position 16 t + lane % 16, dims 32 g + 16 j ..
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
__global__ __launch_bounds__(64 * FEW_WAVES, 2) void paged_few_q8_kernel(
    PagedKv kv, int few_rows, int max_workers, RowsScratch rs, const float *__restrict__ q,
    int part_rows, float *__restrict__ part, int2 *__restrict__ shared, float *__restrict__ out)
{
    extern __shared__ long long before[]; // [seqs + 1]
    __shared__ long long wsum[4];
    if (blockIdx.x * FEW_WAVES >= max_workers) { // one more workgroup: the tile form's plan
        rows_plan(kv, few_rows, rs, (int *)before);
        return;
    }
    const FewPlan plan = few_plan<TILE, SHARED>(kv, few_rows, max_workers, before, wsum);
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x + max_workers / FEW_WAVES *
                                                                  (threadIdx.x >> 6));
    if (w >= plan.workers) return;
    long long at = plan.begin(w);
    const long long stop = plan.begin(w + 1);
    const int rep = kv.heads / kv.kvh;
    const size_t hsize = (size_t)KV_D << kv.shift; // a head's codes of a page
    const size_t psize = 2 * kv.kvh * (hsize / KV_D * kv_row_bytes(KV_T_Q8));
    const int pmask = (1 << kv.shift) - 1;

    int s = 0; // the slot that holds tile `at`: the last with before[s] <= at
    {
        int hi = kv.seqs;
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (before[mid] <= at) s = mid;
            else hi = mid;
        }
    }
    while (at < stop) {
        while (before[s + 1] <= at) ++s; // slots without tiles
        s = __builtin_amdgcn_readfirstlane(s);
        const SlotRows sr = slot_rows(kv, s);
        const int skip = skipped<SHARED>(kv, s, sr);
        const int tiles = slot_tiles<TILE>(sr.len - skip);
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
        const int sees = ok ? sr.len - sr.n + tok : -1; // this row's last visible position
        Query query;
        query.load(q + row * KV_D, ok, g);
        f32x4 acc[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        // m: the running maximum less LIFT; top: a power of two above all scales of
        // values seen (not below 2^-100, that its inverse be one too)
        float m = -INFINITY, l = 0.f, top = 0x1p-100f;

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
                    st.k[t][j] = cached<i32x4, once.value>(kb, (p + c) * KV_D + 32 * g + 16 * j);
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
            __builtin_amdgcn_readfirstlane(mine != below && mine != above) != 0;
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
                // (the power of two above bm)
                const float up = __builtin_bit_cast(
                    float, (__builtin_bit_cast(unsigned, bm) & 0x7f800000u) + 0x00800000u);
                const float tn = bm > top ? up : top;
                // a row that has seen nothing yet keeps zero weights
                const float base = mn == -INFINITY ? 0.f : mn;
                if (__any(mn != m || tn != top)) {
                    const float corr = __builtin_amdgcn_exp2f(m - base);
                    const float both = corr * (top / tn);
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[x] *= both;
                    l *= corr;
                    m = mn;
                    top = tn;
                }
                const float inv = __builtin_bit_cast(
                    float, 0x7f000000u - __builtin_bit_cast(unsigned, top)); // 1 / top
                half8 hi, lo;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(sv[i] - base),
                                p1 = __builtin_amdgcn_exp2f(sv[i + 1] - base);
                    sum += p0 + p1;
                    half2 x, y;
                    split2(p0 * (b[i] * inv), p1 * (b[i + 1] * inv), x, y);
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
        if (t0 == 0 && lane == 0) { // who shares the unit, for the merge
            const long long last = before[s] + (long long)(kh + 1) * tiles - 1;
            const int n = t1 == tiles ? 1 : plan.worker(last) - w + 1;
            shared[(size_t)s * kv.kvh + kh] = make_int2(w, n);
        }
        float *o, f;
        if (t0 == 0 && t1 == tiles && skip == 0) {
            // (a row that saw nothing gives zeros)
            o = out + row * KV_D;
            f = l > 0.f || l != l ? top * (512.f / l) : 0.f;
        } else {
            const long long slot = (long long)w + (long long)s * kv.kvh + kh;
            o = part + ((size_t)slot * part_rows + c) * PAGED_PART;
            if (ok && g == 0) { // (the maximum itself, and weights of at most 1)
                o[0] = m + LIFT;
                o[1] = l * 0x1p-14f;
            }
            o += 4;
            f = top * 0x1p-5f;
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
                        const float *q, int part_rows, float *part, int2 *shared, float *out,
                        void *stream)
{
    const size_t lds = ((size_t)kv.seqs + 1) * 8;
    const dim3 grid(workers / FEW_WAVES + (rs.cap > 0)), block(64 * FEW_WAVES);
    auto kernel = kv.skip ? paged_few_q8_kernel<true> : paged_few_q8_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, block, lds, (hipStream_t)stream, kv, few, workers, rs, q,
                       part_rows, part, shared, out);
    return (int)hipGetLastError();
}

} // namespace hyq
