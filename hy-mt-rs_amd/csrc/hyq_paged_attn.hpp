// What the two forms of the paged attention share: the slots' rows, the plan of
// the tile form (made by a workgroup of the few-row form's launch) and the
// layout of its scratch.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged.hpp"
#include "hyq_paged_pieces.hpp"
#include "hyq_wave.hpp"

namespace hyq {

// A partial row: maximum, exp-sum, two words unused, 128 sums.
constexpr int PAGED_PART = 132;

// A slot's new rows and length, as its tables say, cut to what can be held:
// rows [begin, begin + n) of the packed ones, the last of them at position
// len - 1. A slot that claims more new rows than positions has rows at
// negative positions, which see nothing.
struct SlotRows {
    int begin, n, len;
};
__device__ __forceinline__ SlotRows slot_rows(const PagedKv &kv, int s)
{
    SlotRows r;
    r.begin = min(max(kv.start[s], 0), kv.rows);
    r.n = min(max(kv.start[s + 1], r.begin), kv.rows) - r.begin;
    r.len = (int)min((long long)max(kv.len[s], 0), (long long)kv.stride << kv.shift);
    return r;
}

// The power of two that a row of queries whose largest is mx is divided by
// before it is split into f16 parts. Not below 2^-100, whose inverse, and that of
// 2^-113, is still a number: scores of such queries and f16 keys stay below 2^-76,
// which no weight feels.
__device__ __forceinline__ int query_exponent(float mx)
{
    return mx > 0.f && mx < INFINITY ? max(ilogbf(mx), -100) : 0;
}

// A vector at a uniform base and an unsigned 32-bit element offset (a scalar
// base with a vector offset in the load: no 64-bit address per lane).
template <class V, class T> __device__ __forceinline__ V at(const T *base, unsigned off)
{
    return *reinterpret_cast<const V *>(reinterpret_cast<const char *>(base) +
                                        (unsigned)(off * sizeof(T)));
}

// x / y for 0 <= x, 1 <= y: 32-bit division where it serves.
__device__ __forceinline__ int divide(long long x, int y)
{
    return x >> 31 ? (int)(x / y) : (int)((unsigned)x / (unsigned)y);
}

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
// Two values' high and low f16 parts, both rounded to nearest: hi, and
// x - hi (exact in f32) by one mixed-precision fma each.
// (The low part is taken from the high one as it is: written as a difference, the
// compiler forms the high part twice, once of an unrounded product, and a value
// near the middle of two f16 loses its low part.)
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

// ---- scales of 8-bit values ----
// A weight p and the scale b of its position become f16 parts of p b, over `top`, a
// power of two above all scales b that the row has seen. Its logarithm is taken off
// p's exponent, up to Q8_LOG_MOST: beyond it p would fall below f32's normal numbers,
// where the exponential is zero (at 2^122 each weight below 2^-18 of the largest). The
// rest is taken off b.
constexpr float Q8_LOG_MOST = 32.f, Q8_MOST = 0x1p32f;
// Partial rows hold weights of at most 2^-24, so that the sum of 2^24 positions'
// values is not beyond the largest of them.
constexpr float Q8_DOWN = 24.f;
__device__ __forceinline__ float q8_rest(float top) { return fminf(Q8_MOST / top, 1.f); }
// A new `top`, where a scale b passes the old one, and what the sums of weights and of
// values over it are to be multiplied with.
struct Q8Top {
    float weights, sums;
};
__device__ __forceinline__ Q8Top q8_top(float b, float &top, float &log_top)
{
    Q8Top to{1.f, 1.f};
    if (b > top) {
        const unsigned up = (__builtin_bit_cast(unsigned, b) & 0x7f800000u) + 0x00800000u;
        const float was = fminf(top, Q8_MOST);
        to.sums = top / __builtin_bit_cast(float, up);
        top = __builtin_bit_cast(float, up);
        to.weights = was / fminf(top, Q8_MOST);
        log_top = fminf((float)((int)(up >> 23) - 127), Q8_LOG_MOST);
    }
    return to;
}

// ---- the few-row form's plan ----
constexpr int FEW_WAVES = 4;

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
template <int TILE> __device__ __forceinline__ int slot_tiles(int positions)
{
    return max(1, (positions + TILE - 1) / TILE);
}
template <int TILE> __device__ __forceinline__ int few_tiles(const PagedKv &kv, int s, int few_rows)
{
    const SlotRows r = slot_rows(kv, s);
    return r.n > 0 && r.n <= few_rows ? slot_tiles<TILE>(r.len) : 0;
}

// before[s], in LDS: the tiles of the slots before s over all KV heads, with
// the total at before[seqs]. 256 threads. (Every workgroup forms it for itself:
// a launch before this one would cost more than the few loads and barriers.)
template <int TILE>
__device__ __forceinline__ FewPlan few_plan(const PagedKv &kv, int few_rows, int max_workers,
                                            long long *before, long long *wsum)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    long long carry = 0;
    for (int b = 0; b < kv.seqs; b += 256) {
        const int s = b + t;
        const long long mine = s < kv.seqs ? (long long)few_tiles<TILE>(kv, s, few_rows) * kv.kvh : 0;
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

// A vector of the cache: ONCE, of pages that one slot reads, not to be kept in the
// caches, which the rows and parts of this launch and the next ones are for.
template <class V, bool ONCE, class T>
__device__ __forceinline__ V cached(const T *base, unsigned off)
{
    const V *p = reinterpret_cast<const V *>(reinterpret_cast<const char *>(base) +
                                             (unsigned)(off * sizeof(T)));
    return ONCE ? __builtin_nontemporal_load(p) : *p;
}

// ---- the tile form's plan ----
constexpr int PR_ROWS = 128;        // query rows per workgroup
constexpr int PR_TILE = 64;         // positions per step
constexpr int PR_FILL = 256;        // workgroups that fill the GPU: one per CU
constexpr int PR_MIN_TILES = 2;     // the shortest piece worth its partial rows

// A block of a slot's new tokens, and what its pieces left.
struct Block {
    int row, toks;    // its first packed row and its tokens
    int part, pieces; // its first partial block and its pieces
};
struct Plan {
    int blocks, groups;
};

// Pieces that fill the GPU with kvh workgroups each (at least one).
__host__ __device__ inline int fill_pieces(int kvh) { return PR_FILL > kvh ? PR_FILL / kvh : 1; }
inline int max_blocks(int seqs, int rows, int tq) { return rows / tq + std::min(seqs, rows); }
// Pieces: at most fill_pieces cuts. A block that is cut c times leaves c + 1 <=
// 2 c parts. Groups: a piece each, or fill_pieces.
inline int max_pieces(int blocks, int kvh) { return blocks + fill_pieces(kvh); }
inline int max_parts(int kvh) { return 2 * fill_pieces(kvh); }
// Workgroups of the merge: `each` of a slot and one per MERGE_ROWS rows of a
// block, for every KV head. (Rows: three prompts beside 27 sessions took 155.1 us
// with 8 and 152.9 with 16 and 32, one prompt 45.3, 44.8 and 45.4.)
constexpr int MERGE_ROWS = 16;
inline long long merge_groups(int seqs, int kvh, int each, int cap)
{
    return ((long long)seqs * each + (long long)cap * (PR_ROWS / MERGE_ROWS)) * kvh;
}

// Where in the scratch the plan's parts lie.
struct RowsScratch {
    Plan *plan;
    Block *blocks;
    Piece *pieces;
    int *groups; // a workgroup's first piece; one more entry than groups
    float *parts;
    int tq, cap; // tokens of a block, blocks there is room for (0: no tile form)
    int most;    // new rows of a slot at most; those of more are not computed
    const int *list; // prefixes: the blocks' packed rows
};
struct RowsLayout {
    size_t blocks, pieces, groups, parts, bytes;
};
inline RowsLayout rows_layout(int seqs, int kvh, int heads, int rows)
{
    const int nb = max_blocks(seqs, rows, PR_ROWS / (heads / kvh));
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    RowsLayout r;
    r.blocks = up(sizeof(Plan));
    r.pieces = r.blocks + up(nb * sizeof(Block));
    r.groups = r.pieces + up(max_pieces(nb, kvh) * sizeof(Piece));
    r.parts = r.groups + up((max_pieces(nb, kvh) + 1) * sizeof(int));
    r.bytes = r.parts + up((size_t)max_parts(kvh) * kvh * PR_ROWS * PAGED_PART * 4);
    return r;
}

__device__ __forceinline__ int block_tiles(const SlotRows &r, int b, int tq)
{
    const int last = r.len - r.n + min(r.n, (b + 1) * tq); // one past the last position seen
    return max(1, (last + PR_TILE - 1) / PR_TILE);
}

// Exclusive scan of one value per thread over 256 threads; returns the total.
__device__ __forceinline__ int scan256(int mine, int &before, int *wsum)
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
    for (int w = 0; w < 4; ++w) {
        if (w < wave) base += wsum[w];
        all += wsum[w];
    }
    before = base + v - mine;
    return all;
}

// The plan, by one workgroup of 256 threads. first: LDS of seqs ints. (The tile
// form's launch waits for it: a round of up to 256 blocks is read and counted
// once, and its scans are few.)
__device__ __forceinline__ void rows_plan(const PagedKv &kv, int few_rows, const RowsScratch &rs,
                                          int *first)
{
    constexpr int TRIES = 16;
    __shared__ int wsum[4];
    __shared__ int sums[TRIES], steps[256];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, tq = rs.tq;
    if (t < TRIES) sums[t] = 0;
    int count = 0;
    for (int b = 0; b < kv.seqs; b += 256) {
        int nb = 0, before;
        if (b + t < kv.seqs) {
            const SlotRows r = slot_rows(kv, b + t);
            nb = r.n > few_rows && r.n <= rs.most ? (r.n + tq - 1) / tq : 0;
        }
        const int all = scan256(nb, before, wsum);
        if (b + t < kv.seqs) first[b + t] = count + before;
        count += all;
    }
    // (starts that do not ascend could claim rows twice: what the scratch has
    // no room for is left out)
    count = min(count, rs.cap);
    __syncthreads();
    // block b, where there is one: its slot, rows and steps (0: none)
    struct At {
        int s, x;
        SlotRows r;
    };
    auto block_at = [&](int b) {
        At a{};
        if (b >= count) return a;
        int hi = kv.seqs; // the last slot with first[s] <= b
        while (hi - a.s > 1) {
            const int mid = (a.s + hi) >> 1;
            if (first[mid] <= b) a.s = mid;
            else hi = mid;
        }
        a.r = slot_rows(kv, a.s);
        a.x = block_tiles(a.r, b - first[a.s], tq);
        return a;
    };
    const At a0 = block_at(t);
    // all steps of one KV head, and the longest block's (a block has at most
    // 2^24 / 64 steps, so that 256 of them fit an int)
    long long tiles = 0;
    int before0 = 0, longest = a0.x;
    for (int b = 0; b < count; b += 256) {
        const int x = b ? block_at(b + t).x : a0.x;
        int before;
        tiles += scan256(x, before, wsum);
        if (b == 0) before0 = before;
        longest = max(longest, x);
    }
    // Two ways to cut. A workgroup per piece, every block in equal pieces of at
    // most `each` steps: the least length, of sixteen, with which the pieces
    // number no more than fill the GPU once (a second round of a few would take
    // as long as the first), or `most`, of which that is sure unless the blocks
    // alone are many. Or, where that leaves the longest piece more than
    // GROUP_COST steps above the mean, the blocks' steps in sequence in equal
    // shares, a workgroup going through the pieces of its share (it begins and
    // ends each, which takes about as long as GROUP_COST steps). Equal pieces and
    // shares: one slot's 16 even blocks 46.2 and 53.5 us, three uneven prompts
    // beside 27 sessions 173.3 and 169.6.
    constexpr int GROUP_COST = 4;
    const int fill = fill_pieces(kv.kvh), room = max(fill - count, (fill + 1) / 2);
    const int least = max(PR_MIN_TILES, divide(tiles + fill - 1, fill));
    const int most = max(PR_MIN_TILES, divide(tiles + room - 1, room));
    auto length = [&](int i) { return least + divide((long long)(most - least) * i, TRIES - 1); };
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o, 64));
    // a length for each of 16 threads, a sixteenth of a round's blocks for each
    // 16 threads
    const int mine = length(t & (TRIES - 1));
    int tried = 0;
    for (int b = 0; b < count; b += 256) {
        __syncthreads(); // (the last round's readers, and wsum's)
        steps[t] = b ? block_at(b + t).x : a0.x;
        __syncthreads();
        for (int i = t / TRIES; i < min(count - b, 256); i += 256 / TRIES)
            tried += (unsigned)(steps[i] + mine - 1) / (unsigned)mine;
    }
    atomicAdd(sums + (t & (TRIES - 1)), tried);
    if (lane == 0) wsum[wave] = longest;
    __syncthreads();
    longest = max(max(wsum[0], wsum[1]), max(wsum[2], wsum[3]));
    tried = sums[lane & (TRIES - 1)];
    const unsigned fits = (unsigned)__ballot(tried <= fill) & 0xffffu;
    const int each = fits ? length(__ffs((int)fits) - 1) : most;
    const bool shares = !fits || min(each, longest) > least + GROUP_COST;
    int npieces = 0, nparts = 0;
    long long done = 0; // steps before this round's blocks
    for (int b = 0; b < count; b += 256) {
        const At a = b ? block_at(b + t) : a0;
        int xbefore = before0, before, k = 0, share = 0;
        const int xall = b || count > 256 ? scan256(a.x, xbefore, wsum) : 0;
        const long long at = done + xbefore; // the block's first step in the sequence
        done += xall;
        if (a.x) {
            share = divide(at, least);
            k = shares ? divide(at + a.x - 1, least) - share + 1
                       : (int)((unsigned)(a.x + each - 1) / (unsigned)each);
        }
        // pieces and parts by one scan: both below 2^15 in a round
        const int all = scan256(k | (k > 1 ? k : 0) << 16, before, wsum);
        if (a.x) {
            const int index = b + t - first[a.s], part = nparts + (before >> 16);
            rs.blocks[b + t] = Block{a.r.begin + index * tq, min(tq, a.r.n - index * tq), part, k};
            for (int i = 0; i < k; ++i) {
                const int piece = npieces + (before & 0xffff) + i;
                int t0, t1;
                if (shares) {
                    const long long from = (long long)(share + i) * least;
                    t0 = (int)max(0ll, from - at);
                    t1 = (int)min((long long)a.x, from + least - at);
                    if (at + t0 == from) rs.groups[share + i] = piece;
                } else {
                    t0 = divide((long long)a.x * i, k);
                    t1 = divide((long long)a.x * (i + 1), k);
                    rs.groups[piece] = piece;
                }
                rs.pieces[piece] = Piece{a.s,       index,   t0,    t1, k > 1 ? part + i : -1,
                                         a.r.begin, a.r.n, a.r.len - a.r.n};
            }
        }
        npieces += all & 0xffff;
        nparts += all >> 16;
    }
    if (t == 0) {
        const int groups = shares ? divide(tiles + least - 1, least) : npieces;
        rs.groups[groups] = npieces;
        *rs.plan = Plan{count, groups};
    }
}

// ---- prefixes that several slots share ----
// A group's slots have their first `skip` positions in common, on the same pages.
// The tokens of the group's slots stand in blocks in `list`, each slot in as many
// places as the group's widest, so that none lies in two blocks, and their query
// rows see those positions whole. Blocks of 16 rows are attended by the few-row form
// beside the slots' own positions (narrow), where they are many blocks of 128 rows by
// the tile form in a launch of its own, both from the first slot's table row. They
// leave parts that the merge joins with the slots' own. The plan lists the pieces of
// both forms, one of a block or a slot and of one KV head for a worker of the few-row
// form.
// Two waves on each SIMD, and one for f32 pages. The few-row form's launch beside 64 slots
// that share 8192 positions of f16 pages, and beside four groups of 24 that share 3100 of
// 8-bit ones, us: 25 and 41 with 1024, 19 and 38 with 1536, 18 and 31 with 2048, 22 and 36
// with three waves. Four layers of eight slots over 3000 positions, of f32 pages, 117 us
// with 2048 and 92 with 1024.
constexpr int FEW_PIECES = 2048;
__host__ __device__ inline int few_pieces(int type)
{
    return type == KV_T_F32 ? FEW_PIECES / 2 : FEW_PIECES;
}
// (a slot and KV head has a piece at least)
inline int shared_cap(int seqs)
{
    // (a group has two slots or more, a block of the tile form eight or more but for
    // its last one)
    return seqs / 8 + seqs / 2 + 1;
}
inline int few_most(int seqs, int kvh)
{
    constexpr int LOT = 256 * FEW_WAVES; // (whole ones: a workgroup on each CU)
    return (FEW_PIECES + (seqs + shared_cap(seqs)) * kvh + LOT - 1) / LOT * LOT;
}
struct SharedHead {
    Plan plan;   // blocks, their pieces (as groups)
    int workers; // of the few-row form, a piece each
    int narrow;  // blocks of 16 rows
};
struct SharedPlan {
    SharedHead *head;
    int *leader; // [seqs] the first slot of its group, -1: it can be in none
    int *run;    // [seqs] pages that it has in common with that one
    int *skip;   // [seqs] positions that the slot's group attends, 0: none
    SharedPlace *place; // [seqs]
    FewPiece *few;      // [few_most]
    int *list;          // [cap * tq] packed rows, -1 where none
    Piece *pieces;      // [most]
    int tq, cap, most, few_most;
    __device__ __forceinline__ PlanSizes sizes(const PagedKv &kv) const
    {
        return PlanSizes{kv.seqs, kv.kvh, kv.rows, kv.stride, kv.shift, tq, cap, most, few_most};
    }
};
struct SharedLayout {
    size_t ints, place, few, list, pieces, bytes;
    int cap, most;
};
inline SharedLayout shared_layout(int seqs, int kvh, int heads)
{
    const int tq = PR_ROWS / (heads / kvh);
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    SharedLayout l;
    l.cap = shared_cap(seqs);
    l.most = l.cap + fill_pieces(kvh);
    l.ints = up(sizeof(SharedHead));
    l.place = l.ints + up((size_t)seqs * 4) * 3;
    l.few = l.place + up((size_t)seqs * sizeof(SharedPlace));
    l.list = l.few + up((size_t)few_most(seqs, kvh) * sizeof(FewPiece));
    l.pieces = l.list + up((size_t)l.cap * tq * 4);
    l.bytes = l.pieces + up((size_t)l.most * sizeof(Piece));
    return l;
}
inline SharedPlan shared_plan(const void *plan, int seqs, int kvh, int heads)
{
    const SharedLayout l = shared_layout(seqs, kvh, heads);
    char *base = (char *)const_cast<void *>(plan);
    const size_t each = ((size_t)seqs * 4 + 255) / 256 * 256;
    SharedPlan p;
    p.head = (SharedHead *)base;
    p.skip = (int *)(base + l.ints);
    p.leader = (int *)(base + l.ints + each);
    p.run = (int *)(base + l.ints + 2 * each);
    p.place = (SharedPlace *)(base + l.place);
    p.few = (FewPiece *)(base + l.few);
    p.list = (int *)(base + l.list);
    p.pieces = (Piece *)(base + l.pieces);
    p.tq = PR_ROWS / (heads / kvh);
    p.cap = l.cap;
    p.most = l.most;
    p.few_most = few_most(seqs, kvh);
    return p;
}
inline size_t shared_parts_bytes(int seqs, int kvh, int heads)
{
    return (size_t)shared_layout(seqs, kvh, heads).most * kvh * PR_ROWS * PAGED_PART * 4;
}
// A worker's piece, cut to what there is.
template <int TILE>
__device__ __forceinline__ FewPiece few_piece(const PagedKv &kv, const SharedPlan &sp, int w)
{
    return cut_few_piece(sp.sizes(kv), TILE, sp.few[w]);
}

// hyq_paged_few.hip: slots of at most `few` <= paged_few_rows(heads / kv_heads)
// new rows, with the plan where there is a tile form; and the merge of both.
int paged_few_rows(int rep);
size_t paged_few_scratch(int type, bool shared, int seqs, int kvh, int heads, int few);
// (sp, and the prefixes' parts: null where there is no plan of shared prefixes)
int launch_paged_few(const PagedKv &kv, int few, const RowsScratch &rs, const SharedPlan *sp,
                     const float *q, float *part, float *out, void *stream);
int launch_paged_merge(const PagedKv &kv, int few, const RowsScratch &rs, const SharedPlan *sp,
                       const float *part, const float *prefix, float *out, void *stream);
// hyq_paged_few_q8.hip: the few-row form of 8-bit pages, as launch_paged_few has
// laid it out.
int launch_paged_few_q8(const PagedKv &kv, int few, int workers, const RowsScratch &rs,
                        const SharedPlan *sp, const float *q, int part_rows, float *part,
                        int2 *shared, float *out, void *stream);
// hyq_paged_rows.hip: the slots of more.
int launch_paged_rows(const PagedKv &kv, const RowsScratch &rs, const float *q, float *out,
                      void *stream);
// The shared prefixes, to parts.
int launch_paged_prefix(const PagedKv &kv, const SharedPlan &sp, const float *q, float *parts,
                        void *stream);

} // namespace hyq
