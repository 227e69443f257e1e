// Which slots of a step share their first pages, and what the attention does for
// them once: the plan of hyq_paged_shared_attention_d, made on the device.
//
// A launch of one workgroup per slot finds the first slot of its group and counts
// the entries that both tables have in common. A second launch takes of every
// group the prefix that saves most, sum over its slots but one of the prefix's
// pages, gives the slots that have it their places in blocks, and cuts the blocks'
// steps into pieces that fill the GPU once. Everything is whole numbers, and every
// slot's place follows from the slots before it, so the plan does not depend on
// the order in which threads run.
//
// Bound by loads that wait for each other and by barriers (the waves of the first launch
// wait 90 % of their cycles, of the second 71): 14 us for eight slots, 18 for 64, 19 for
// 105, 24 for 256, once a step, not a layer. Then by the counts, which compare each
// slot's key with those of all slots, in every workgroup: 37 us for 512, 91 for 1024,
// 1040 for 4096. A layer of 64 slots over 8200 positions in common and 300 of their own,
// 32 heads over 8, f16 pages: 51 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged_attn.hpp"

namespace hyq {

namespace {

// What a slot shares by: its group's number or its first page; -1 where it has more
// than few new rows or none, or no whole page before them.
struct Candidate {
    int key, pages; // pages: whole ones before the new rows
};
__device__ __forceinline__ Candidate candidate(const PagedKv &kv, const int *group, int s, int few)
{
    const SlotRows r = slot_rows(kv, s);
    Candidate c{-1, max(r.len - r.n, 0) >> kv.shift};
    if (r.n < 1 || r.n > few || c.pages < 1) return c;
    const int page = kv.table[(size_t)s * kv.stride];
    if ((unsigned)page < (unsigned)kv.npages) c.key = group ? group[s] : page;
    return c;
}

// Grid: a workgroup per slot.
__global__ __launch_bounds__(256) void shared_runs_kernel(PagedKv kv, const int *__restrict__ group,
                                                          int few, int *__restrict__ leader,
                                                          int *__restrict__ run)
{
    __shared__ int first, end;
    const int s = blockIdx.x, t = threadIdx.x;
    const Candidate c = candidate(kv, group, s, few);
    if (t == 0) first = s;
    __syncthreads();
    if (c.key >= 0)
        for (int b = t; b < s; b += 256)
            if (candidate(kv, group, b, few).key == c.key) {
                atomicMin(&first, b);
                break;
            }
    __syncthreads();
    const int lead = first;
    int pages = c.key < 0 ? 0 : c.pages;
    if (c.key >= 0 && lead != s) {
        pages = min(pages, candidate(kv, group, lead, few).pages);
        const int *a = kv.table + (size_t)s * kv.stride, *b = kv.table + (size_t)lead * kv.stride;
        // (as many at once as the first slots' tables are long: one round in most)
        for (int i = 0; i < pages; i += 256) {
            __syncthreads();
            if (t == 0) end = pages;
            __syncthreads();
            const int e = i + t;
            if (e < pages && (a[e] != b[e] || (unsigned)a[e] >= (unsigned)kv.npages))
                atomicMin(&end, e);
            __syncthreads();
            if (end < min(i + 256, pages)) {
                pages = end;
                break;
            }
        }
    }
    if (t == 0) {
        leader[s] = c.key < 0 ? -1 : lead;
        run[s] = pages;
    }
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
    int u = wsum[lane & 15]; // the waves' sums, summed by each 16 lanes
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const int x = __shfl_up(u, o, 16);
        if ((lane & 15) >= o) u += x;
    }
    before = v - mine + (wave ? __builtin_amdgcn_readlane(u, wave - 1) : 0);
    return __builtin_amdgcn_readlane(u, 15);
}

// What the i-th of k pieces takes of x tiles or steps: the first x % k one more.
__device__ __forceinline__ int2 share(int x, int i, int k)
{
    const int q = (int)((unsigned)x / (unsigned)k), more = x - q * k, from = i * q + min(i, more);
    return make_int2(from, from + q + (i < more));
}
// The last of n ascending numbers that is at most x (the first is).
__device__ __forceinline__ int last_of(const int *a, int n, int x)
{
    int s = 0;
    while (n - s > 1) {
        const int mid = (s + n) >> 1;
        if (a[mid] <= x) s = mid;
        else n = mid;
    }
    return s;
}
__device__ __forceinline__ int pieces_of(int tiles, int piece)
{
    return (int)((unsigned)(tiles + piece - 1) / (unsigned)piece);
}

// What the plan knows of its slots and blocks, in LDS.
struct PlanLds {
    unsigned *key; // [seqs], in whole fours: the group's first slot << 20 | pages in common
    int *ways;     // (where `key` was) a slot's pieces
    unsigned long long *best; // [seqs] of a group's first slot: saving, pages
    int *begin, *len;         // (where `best` was) the slot's rows, its positions
    int *pages;  // the group's slots with as many pages in common; then those it attends
    int *first;  // of a group's first slot: its slots, its first block; then a slot's first worker
    int *wide;   // new rows of the group's slots at most
    unsigned *steps;     // [cap] a block's steps
    int *part;           // [cap + 1] its first part
    int *rank;           // the slot's place in its group, then in its block
    short *block;        // and that
    short *of;           // [cap] a block's group
    unsigned char *rows; // new rows of the slot
    unsigned char *toks; // [cap] a block's tokens
    static size_t bytes(int n, int cap)
    {
        return (size_t)((n + 3) & ~3) * 4 + (size_t)n * 27 + (size_t)cap * 11 + 4;
    }
    __device__ PlanLds(void *at, int n, int cap)
    {
        key = (unsigned *)at, ways = (int *)at, begin = (int *)(key + ((n + 3) & ~3));
        best = (unsigned long long *)begin, len = begin + n, pages = len + n, first = pages + n;
        wide = first + n, rank = wide + n, steps = (unsigned *)(rank + n);
        part = (int *)(steps + cap), block = (short *)(part + cap + 1), of = block + n;
        rows = (unsigned char *)(of + cap), toks = rows + n;
    }
    // Adds to into[s], for the slots s of 64 lanes and by 16 waves a share of the keys
    // each, those of [0, end) of the group of `from` that have as many pages in common.
    __device__ __forceinline__ void count(unsigned from, int end, int *into) const
    {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        const unsigned room = 0xfffffu - (from & 0xfffffu);
        int n = 0;
#pragma unroll 1
        for (int b = 4 * (threadIdx.x >> 6); b < end; b += 64) {
            const u32x4 k = *(const u32x4 *)(key + b);
#pragma unroll
            for (int i = 0; i < 4; ++i) n += b + i < end && k[i] - from <= room;
        }
        if (n) atomicAdd(into, n);
    }
};

// PLAN_GROUPS workgroups, each of which makes the whole plan for itself; the first
// one writes it, but for the few-row form's pieces, of which each writes some (64 slots
// 14.3 us, and 15.4 where one workgroup wrote them all; 105 slots 16.5 and 17.9). Their
// time is that of their barriers and of their code, which they find in no cache: what
// they need is read once, numbers are 32 bits, and few loops are unrolled.
constexpr int PLAN_GROUPS = 8;
// The tiles of narrow blocks, over all KV heads, up to which they take less time than
// the tile form, in steps of 16 positions, and of 32 in 8-bit pages. Narrow and wide, us
// a layer, 16 heads over 4 and 32 over 8: f16 pages at 3008 tiles 22.0 and 24.9, at 4000
// 27.7 and 26.3, at 8064 33.2 and 30.9; f32 ones at 4000 24.0 and 28.8, 6016 27.4 and
// 29.6, 8032 31.5 and 31.6, 16000 55.9 and 38.2; 8-bit ones at 4096 26.7 and 29.1, 8064
// 32.4 and 32.6, 16000 41.7 and 38.1. (f32's limit lies before its crossing, at some 8000:
// between them wide blocks take up to 2 us more.)
__device__ __forceinline__ int most_narrow_tiles(int type)
{
    return type == KV_T_Q8 ? 8192 : type == KV_T_F16 ? 3500 : 6500;
}
__global__ __launch_bounds__(1024) void shared_plan_kernel(PagedKv kv, int few,
                                                           long long worth, SharedPlan sp)
{
    extern __shared__ __align__(16) unsigned lds[];
    constexpr int TRIES = 16;
    __shared__ int wsum[16], tried[TRIES];
    // all blocks' steps; the tiles of the few-row form, and its slots and blocks; the
    // groups' saving; the narrow blocks' tiles, and those blocks
    __shared__ unsigned sum[6];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = kv.seqs;
    const PlanLds x(lds, n, sp.cap);
    const bool writes = blockIdx.x == 0;
    constexpr unsigned NONE = 0xfff00000u; // (a group has a page in common at least)
    if (t < 6) sum[t] = 0;
#pragma unroll 1
    for (int s = t; s < ((n + 3) & ~3); s += 1024) {
        const int l = s < n ? sp.leader[s] : -1;
        x.key[s] = l < 0 ? NONE : (unsigned)l << 20 | (unsigned)sp.run[s];
        if (s >= n) break;
        const SlotRows r = slot_rows(kv, s);
        x.best[s] = 0;
        x.rows[s] = (unsigned char)(r.n <= few ? r.n : 0);
        x.first[s] = x.wide[s] = x.pages[s] = x.rank[s] = 0;
    }
    __syncthreads();
    // the saving of a prefix as long as each slot's run, and the largest of a group
#pragma unroll 1
    for (int s = lane; s < n; s += 64)
        if (x.key[s] != NONE) x.count(x.key[s], n, x.pages + s);
    __syncthreads();
#pragma unroll 1
    for (int s = t; s < n; s += 1024) {
        const unsigned key = x.key[s], run = key & 0xfffffu;
        const int others = run ? x.pages[s] - 1 : 0;
        if (others > 0)
            atomicMax(x.best + (key >> 20), (unsigned long long)others * run << 24 | run);
    }
    __syncthreads();
    // (a group's at most 2^20, of 2048 at most)
#pragma unroll 1
    for (int s = t; s < n; s += 1024)
        if (x.best[s]) atomicAdd(&sum[3], min((unsigned)(x.best[s] >> 24), 1u << 20));
    __syncthreads();
    const bool shares = ((long long)sum[3] << kv.shift) * kv.kvh >= worth;
    // a slot's place among its group's, the group's slots and its widest one's tokens
    auto pages_of = [&](unsigned key) {
        const unsigned run = key & 0xfffffu;
        const unsigned pages = run && shares ? (unsigned)x.best[key >> 20] & 0xffffffu : 0;
        return run >= pages ? pages : 0;
    };
#pragma unroll 1
    for (int s = lane; s < n; s += 64) {
        const unsigned key = x.key[s], pages = pages_of(key);
        if (pages) x.count((key & NONE) | pages, s, x.rank + s);
    }
#pragma unroll 1
    for (int s = t; s < n; s += 1024) {
        const unsigned l = x.key[s] >> 20, pages = pages_of(x.key[s]);
        x.pages[s] = (int)pages;
        if (writes) sp.skip[s] = (int)(pages << kv.shift);
        if (!pages) continue;
        atomicAdd(x.first + l, 1);
        atomicMax(x.wide + l, (int)x.rows[s]);
    }
    __syncthreads();
    const int tile = kv.type == KV_T_Q8 ? 5 : 4; // (the few-row form's step, as a logarithm)
    auto tiles = [&](int positions) { return max(1, (positions + (1 << tile) - 1) >> tile); };
#pragma unroll 1
    for (int s = t; s < n; s += 1024)
        if (x.first[s]) {
            const int each = few / x.wide[s], mine = pieces_of(x.first[s], each);
            atomicAdd(&sum[4],
                      min((unsigned)mine * (unsigned)tiles(x.pages[s] << kv.shift), 1u << 20));
            atomicAdd(&sum[5], (unsigned)mine);
        }
    __syncthreads();
    // (and where they are no more than there is room for: blocks of one slot each, as with
    // nine query heads or more to a KV head, may be)
    const int most_narrow = most_narrow_tiles(kv.type);
    const bool narrow = (long long)sum[4] * kv.kvh <= most_narrow && (int)sum[5] <= sp.cap;
    const int tq = narrow ? few : sp.tq;
    int blocks = 0;
#pragma unroll 1
    for (int b = 0; b < n; b += 1024) {
        const int s = b + t, slots = s < n ? x.first[s] : 0;
        const int each = slots ? tq / x.wide[s] : 1, mine = (slots + each - 1) / each;
        int before;
        const int all = scan1024(mine, before, wsum);
        const int first = blocks + before;
#pragma unroll 1
        for (int i = 0; i < mine && first + i < sp.cap; ++i) {
            const int positions = x.pages[s] << kv.shift;
            const unsigned steps = narrow ? tiles(positions) : (positions + PR_TILE - 1) / PR_TILE;
            x.of[first + i] = (short)s;
            x.steps[first + i] = steps;
            x.toks[first + i] = (unsigned char)(min(each, slots - i * each) * x.wide[s]);
            atomicAdd(&sum[0], steps);
        }
        if (s < n) x.first[s] = first;
        blocks += all;
    }
    blocks = min(blocks, sp.cap);
    __syncthreads();
    // the slots' places in the blocks, and what their own positions are
    auto tiles_of = [&](int s) {
        return x.rows[s] ? tiles(x.len[s] - (x.pages[s] << kv.shift)) : 0;
    };
#pragma unroll 1
    for (int s = t; s < n; s += 1024) {
        const SlotRows r = slot_rows(kv, s);
        x.begin[s] = r.begin;
        x.len[s] = r.len;
        const int own = tiles_of(s);
        if (own) {
            atomicAdd(&sum[1], (unsigned)min(own, (1 << 20) - 1));
            atomicAdd(&sum[2], 1u);
        }
        if (!x.pages[s]) continue;
        const int l = (int)(x.key[s] >> 20), wide = x.wide[l], each = tq / wide;
        const int up = x.rank[s] / each, at = (x.rank[s] - up * each) * wide;
        const int b = min(x.first[l] + up, sp.cap - 1);
#pragma unroll 1
        for (int i = 0; writes && i < wide; ++i)
            sp.list[b * tq + at + i] = i < x.rows[s] ? x.begin[s] + i : -1;
        x.block[s] = (short)b;
        x.rank[s] = at; // (its first token's place in the block)
    }
    int parts = 0;
    if (!narrow) {
        // Pieces of at most `each` steps: the least, of sixteen lengths, with which they
        // number no more than fill the GPU once, or the last one, of which that is sure
        // unless the blocks alone are many.
        const int total = (int)sum[0], fill = fill_pieces(kv.kvh);
        const int room = max(fill - blocks, (fill + 1) / 2);
        const int least = max(PR_MIN_TILES, (total + fill - 1) / fill);
        const int most = max(least, (total + room - 1) / room);
        const int more = (most - least + TRIES - 2) / (TRIES - 1);
        int pieces = 0;
#pragma unroll 1
        for (int b = lane; b < blocks; b += 64)
            pieces += pieces_of((int)x.steps[b], least + more * wave);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) pieces += __shfl_xor(pieces, o, 64);
        if (lane == 0) tried[wave] = pieces;
        __syncthreads();
        const unsigned fits = (unsigned)__ballot(tried[lane & (TRIES - 1)] <= fill) & 0xffffu;
        const int each = least + more * (fits ? __ffs((int)fits) - 1 : TRIES - 1);
#pragma unroll 1
        for (int b = 0; b < blocks; b += 1024) {
            const int at = b + t, steps = at < blocks ? (int)x.steps[at] : 0;
            int before;
            const int all = scan1024(pieces_of(steps, each), before, wsum);
            if (at < blocks) x.part[at] = parts + before;
            parts += all;
        }
        if (t == 0) x.part[blocks] = parts;
        __syncthreads();
#pragma unroll 1
        for (int p = t; writes && p < parts; p += 1024) {
            const int b = last_of(x.part, blocks, p), s = x.of[b];
            const int2 by = share((int)x.steps[b], p - x.part[b], x.part[b + 1] - x.part[b]);
            sp.pieces[p] = Piece{s, b, by.x, by.y, p, 0, x.toks[b], x.pages[s] << kv.shift};
        }
    } else {
        __syncthreads();
    }
    // The slots' own positions, by the few-row form: pieces of at most `piece` tiles, so
    // long that they number as many as few_pieces says. (Each slot's and block's last one
    // is shorter; the matrix unit bounds f32 pages, whose pieces are cut as if there were
    // none. Others, 32 heads over 8, us for two layers in f16 pages of 128 slots over
    // 2000 positions in common and 500 of their own, and of four groups in 8-bit ones:
    // 287 and 176 with half the number at least, 272 and 176 with 5/8, 265 and 176 with
    // 11/16, 264 and 178 with 3/4.)
    const int head = few_pieces(kv.type) / kv.kvh; // of a KV head
    const unsigned units = sum[2] + (narrow ? sum[5] : 0);
    const unsigned all_tiles = sum[1] + (narrow ? sum[4] : 0);
    const int spread = kv.type == KV_T_F32 ? head : max(head - (int)units, head * 11 / 16);
    // (The merge waits for a row's parts: where blocks are narrow, pieces grow with the
    // longest block's tiles, up to four. Eight slots over 600, 1500 and 3000 positions in
    // common, 38, 94 and 188 tiles, 16 heads over 4, us a layer with pieces of 1, 2, 3, 4
    // and 6 tiles at least: f16 pages 14.1 13.5 14.7 16.4 18.3, 18.2 16.1 16.9 17.2 18.0,
    // 27.1 21.0 19.3 19.0 20.5; 32 slots over 1000, 63 tiles, 23.3 23.1 19.9 19.9 21.8. Of
    // few blocks with 49 to 128 tiles two would be the better: the 94 tiles in f32 pages
    // take 15.6 with two and 17.0 with three.)
    int least = 1;
    if (narrow) {
        int longest = 0;
#pragma unroll 1
        for (int b = lane; b < blocks; b += 64) longest = max(longest, (int)x.steps[b]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o, 64));
        least = longest <= 16 ? 1 : longest <= 48 ? 2 : longest <= 128 ? 3 : 4;
    }
    const int piece = max(least, pieces_of((int)min(all_tiles, 0x7fff0000u), spread));
    int workers = 0;
    if (narrow) {
#pragma unroll 1
        for (int b = 0; b < blocks; b += 1024) {
            const int at = b + t, ways = at < blocks ? pieces_of((int)x.steps[at], piece) : 0;
            int before;
            const int all = scan1024(ways * kv.kvh, before, wsum);
            if (at < blocks) x.part[at] = workers + before;
            workers += all;
        }
        __syncthreads();
    }
    const int of_blocks = workers;
#pragma unroll 1
    for (int b = 0; b < n; b += 1024) {
        const int s = b + t, ways = s < n ? pieces_of(tiles_of(s), piece) : 0;
        int before;
        const int all = scan1024(ways * kv.kvh, before, wsum);
        if (s < n) {
            SharedPlace p{x.begin[s], x.rows[s], 0, 0, 0, workers + before, ways, 0};
            if (x.pages[s]) {
                const int at = x.block[s];
                p.part = x.part[at];
                p.pieces = narrow ? pieces_of((int)x.steps[at], piece) : x.part[at + 1] - p.part;
                p.row = x.rank[s] * (kv.heads / kv.kvh);
            }
            if (writes) sp.place[s] = p;
            x.first[s] = workers + before;
            x.ways[s] = ways;
        }
        workers += all;
    }
    workers = min(workers, sp.few_most);
    __syncthreads();
#pragma unroll 1
    for (int w = blockIdx.x * 256 + t; t < 256 && w < workers; w += PLAN_GROUPS * 256) {
        if (w < of_blocks) {
            const int b = last_of(x.part, blocks, w), s = x.of[b];
            const int ways = pieces_of((int)x.steps[b], piece);
            const int kh = (int)((unsigned)(w - x.part[b]) / (unsigned)ways);
            const int2 by = share((int)x.steps[b], w - x.part[b] - kh * ways, ways);
            sp.few[w] = FewPiece{s,         kh,        by.x, by.y, b * tq, x.toks[b],
                                 x.pages[s] << kv.shift, 0,    ways, 1,      {}};
            continue;
        }
        const int s = last_of(x.first, n, w), ways = max(1, x.ways[s]); // (a slot that has pieces)
        const int kh = (int)((unsigned)(w - x.first[s]) / (unsigned)ways);
        const int2 by = share(tiles_of(s), w - x.first[s] - kh * ways, ways);
        sp.few[w] = FewPiece{s,          kh,        by.x,     by.y,
                             x.begin[s], x.rows[s], x.len[s], x.pages[s] << kv.shift,
                             ways,       0,         {}};
    }
    if (writes && t == 0) *sp.head = SharedHead{Plan{blocks, parts}, workers, narrow};
}

} // namespace

int launch_shared_plan(const PagedKv &kv, const int *group, long long least, void *plan,
                       void *stream)
{
    const SharedPlan sp = shared_plan(plan, kv.seqs, kv.kvh, kv.heads);
    const int few = paged_few_rows(kv.heads / kv.kvh);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(shared_runs_kernel, dim3(kv.seqs), dim3(256), 0, st, kv, group, few,
                       sp.leader, sp.run);
    hipLaunchKernelGGL(shared_plan_kernel, dim3(PLAN_GROUPS), dim3(1024),
                       PlanLds::bytes(kv.seqs, sp.cap), st, kv, few, least, sp);
    return (int)hipGetLastError();
}

} // namespace hyq
