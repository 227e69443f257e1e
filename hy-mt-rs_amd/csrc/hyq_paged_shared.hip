// Which slots of a step share their first pages, and what the attention does for
// them once: the plan of hyq_paged_shared_attention_d, made on the device.
//
// A launch of one workgroup per slot finds the first slot of its group and counts
// the entries that both tables have in common. One workgroup then takes of every
// group the prefix that saves most, sum over its slots but one of the prefix's
// pages, numbers the tokens of the slots that have it, and cuts their blocks'
// steps into pieces that fill the GPU once. Everything is whole numbers, and every
// slot's place follows from the slots before it, so the plan does not depend on
// the order in which threads run.
//
// Bound by loads that wait for each other: once a step, not a layer.
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
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        if (w < wave) base += wsum[w];
        all += wsum[w];
    }
    before = base + v - mine;
    return all;
}

// One workgroup.
__global__ __launch_bounds__(1024) void shared_plan_kernel(PagedKv kv, int few, SharedPlan sp)
{
    extern __shared__ unsigned long long best[]; // [seqs] of a group's first slot: saving, pages
    int *lead = (int *)(best + kv.seqs), *run = lead + kv.seqs, *rows = run + kv.seqs,
        *base = rows + kv.seqs; // [seqs] each
    __shared__ int wsum[16];
    const int t = threadIdx.x, n = kv.seqs;
    for (int s = t; s < n; s += 1024) {
        best[s] = 0;
        lead[s] = sp.leader[s];
        run[s] = sp.run[s];
        rows[s] = lead[s] < 0 ? 0 : slot_rows(kv, s).n;
        base[s] = 0;
    }
    __syncthreads();
    // the saving of a prefix as long as each slot's run, and the largest of a group
    for (int s = t; s < n; s += 1024) {
        if (lead[s] < 0 || run[s] < 1) continue;
        int others = -1;
        for (int x = lead[s]; x < n; ++x) others += lead[x] == lead[s] && run[x] >= run[s];
        if (others > 0)
            atomicMax(best + lead[s], (unsigned long long)others * run[s] << 24 | (unsigned)run[s]);
    }
    __syncthreads();
    // the pages that a slot's group attends for it
    auto shares = [&](int s) {
        const int pages = lead[s] < 0 ? 0 : (int)(best[lead[s]] & 0xffffff);
        return pages > 0 && run[s] >= pages ? pages : 0;
    };
    // tokens of every group, at its first slot, and its first block
    for (int s = t; s < n; s += 1024)
        if (shares(s)) atomicAdd(base + lead[s], rows[s]);
    __syncthreads();
    int blocks = 0;
    for (int b = 0; b < n; b += 1024) {
        const int s = b + t;
        const int tokens = s < n ? base[s] : 0, mine = (tokens + sp.tq - 1) / sp.tq;
        int before;
        const int all = scan1024(mine, before, wsum);
        const int first = blocks + before;
        for (int i = 0; i < mine && first + i < sp.cap; ++i)
            sp.blocks[first + i] =
                Block{s, min(sp.tq, tokens - i * sp.tq), 0, shares(s) << kv.shift};
        if (s < n) base[s] = first;
        blocks += all;
    }
    blocks = min(blocks, sp.cap); // (starts that do not ascend could claim rows twice)
    __syncthreads();
    for (int s = t; s < n; s += 1024) {
        const int pages = shares(s);
        int at = 0;
        if (pages) {
            at = base[lead[s]] * sp.tq;
            for (int x = lead[s]; x < s; ++x) at += lead[x] == lead[s] && run[x] >= pages ? rows[x] : 0;
            const int begin = slot_rows(kv, s).begin;
            for (int i = 0; i < rows[s]; ++i)
                if (at + i < sp.cap * sp.tq) sp.list[at + i] = begin + i;
        }
        sp.place[s] = at;
        sp.skip[s] = pages << kv.shift;
    }
    __threadfence_block();
    __syncthreads();
    // Pieces of at most `each` steps, so many that they fill the GPU once beside
    // the blocks' last ones (rounded up, a piece a block more than that at most).
    auto steps_of = [&](int b) { return (sp.blocks[b].pieces + PR_TILE - 1) / PR_TILE; };
    long long steps = 0;
    for (int b = 0; b < blocks; b += 1024) {
        int before;
        steps += scan1024(b + t < blocks ? steps_of(b + t) : 0, before, wsum);
    }
    const int fill = fill_pieces(kv.kvh);
    const int each = max(PR_MIN_TILES, divide(steps + fill - 1, fill));
    int parts = 0;
    for (int b = 0; b < blocks; b += 1024) {
        Block blk{};
        int x = 0, k = 0, before;
        if (b + t < blocks) {
            blk = sp.blocks[b + t];
            x = steps_of(b + t);
            k = (x + each - 1) / each;
        }
        const int all = scan1024(k, before, wsum);
        for (int i = 0; i < k; ++i)
            sp.pieces[parts + before + i] =
                Piece{blk.row, b + t, divide((long long)x * i, k), divide((long long)x * (i + 1), k),
                      parts + before + i, 0, blk.toks, blk.pieces};
        if (k) sp.blocks[b + t] = Block{blk.row, blk.toks, parts + before, k};
        parts += all;
    }
    if (t == 0) *sp.plan = Plan{blocks, parts};
}

} // namespace

int launch_shared_plan(const PagedKv &kv, const int *group, void *plan, void *stream)
{
    const SharedPlan sp = shared_plan(plan, kv.seqs, kv.kvh, kv.heads, kv.rows);
    const int few = paged_few_rows(kv.heads / kv.kvh);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(shared_runs_kernel, dim3(kv.seqs), dim3(256), 0, st, kv, group, few,
                       sp.leader, sp.run);
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(1024), (size_t)kv.seqs * 24, st, kv, few,
                       sp);
    return (int)hipGetLastError();
}

} // namespace hyq
