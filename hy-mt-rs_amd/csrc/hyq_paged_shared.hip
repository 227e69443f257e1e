// Which slots of a step share their first pages, and what the attention does for
// them once: the plan of hyq_paged_shared_attention_d, made on the device.
//
// A launch of one workgroup per slot finds the first slot of its group and counts
// the entries that both tables have in common. One workgroup then takes of every
// group the prefix that saves most, sum over its slots but one of the prefix's
// pages, gives the slots that have it their places in blocks, and cuts the blocks'
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

// One workgroup. A wave takes a slot at a time where others are counted for it.
__global__ __launch_bounds__(1024) void shared_plan_kernel(PagedKv kv, int few, SharedPlan sp)
{
    extern __shared__ unsigned long long best[]; // [seqs] of a group's first slot: saving, pages
    // [seqs] each; base: the group's slots, its first block, then a slot's first worker
    int *run = (int *)(best + kv.seqs), *base = run + kv.seqs;
    short *lead = (short *)(base + kv.seqs);
    unsigned char *rows = (unsigned char *)(lead + kv.seqs), *wide = rows + kv.seqs;
    unsigned *steps = (unsigned *)(best + 3 * kv.seqs); // [cap]
    constexpr int TRIES = 16;
    __shared__ int wsum[16], tried[TRIES];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, n = kv.seqs;
    for (int s = t; s < n; s += 1024) {
        best[s] = 0;
        lead[s] = (short)sp.leader[s];
        run[s] = sp.run[s];
        rows[s] = (unsigned char)(lead[s] < 0 ? 0 : slot_rows(kv, s).n);
        base[s] = 0;
    }
    __syncthreads();
    // the saving of a prefix as long as each slot's run, and the largest of a group
    for (int s = wave; s < n; s += 16) {
        const int l = lead[s], pages = run[s];
        if (l < 0 || pages < 1) continue;
        int others = -1;
        for (int b = l; b < n; b += 64) {
            const int x = min(b + lane, n - 1);
            others += __popcll(__ballot(b + lane < n && lead[x] == l && run[x] >= pages));
        }
        if (lane == 0 && others > 0)
            atomicMax(best + l, (unsigned long long)others * pages << 24 | (unsigned)pages);
    }
    __syncthreads();
    // the pages that a slot's group attends for it
    auto shares = [&](int s) {
        const int pages = lead[s] < 0 ? 0 : (int)(best[lead[s]] & 0xffffff);
        return pages > 0 && run[s] >= pages ? pages : 0;
    };
    // a slot's place among its group's, the group's slots and its widest one's tokens
    for (int s = wave; s < n; s += 16) {
        const int l = lead[s], pages = shares(s);
        int before = 0, all = 0, most = 0;
        if (pages)
            for (int b = l; b < n; b += 64) {
                const int x = min(b + lane, n - 1);
                const bool in = b + lane < n && lead[x] == l && run[x] >= pages;
                before += __popcll(__ballot(in && x < s));
                all += __popcll(__ballot(in));
                most = max(most, in ? (int)rows[x] : 0);
            }
        if (lane == 0) {
            sp.skip[s] = pages << kv.shift;
            sp.place[s].block = before;
        }
        if (l != s || !pages) continue;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
        if (lane == 0) {
            base[s] = all;
            wide[s] = (unsigned char)most;
        }
    }
    __syncthreads();
    int blocks = 0;
    for (int b = 0; b < n; b += 1024) {
        const int s = b + t, slots = s < n ? base[s] : 0;
        const int each = slots ? sp.tq / wide[s] : 1, mine = (slots + each - 1) / each;
        int before;
        const int all = scan1024(mine, before, wsum);
        const int first = blocks + before;
        for (int i = 0; i < mine && first + i < sp.cap; ++i) {
            const int pages = shares(s);
            sp.blocks[first + i] = Block{s, min(each, slots - i * each) * wide[s], 0, 0};
            steps[first + i] = (((unsigned)pages << kv.shift) + PR_TILE - 1) / PR_TILE;
        }
        if (s < n) base[s] = first;
        blocks += all;
    }
    blocks = min(blocks, sp.cap);
    __syncthreads();
    for (int s = t; s < n; s += 1024) {
        if (!shares(s)) continue;
        const int l = lead[s], each = sp.tq / wide[l], rank = sp.place[s].block;
        const int b = min(base[l] + rank / each, sp.cap - 1), at = rank % each * wide[l];
        const int begin = slot_rows(kv, s).begin;
        for (int i = 0; i < wide[l]; ++i)
            sp.list[b * sp.tq + at + i] = i < rows[s] ? begin + i : -1;
        sp.place[s].row = at * (kv.heads / kv.kvh);
        sp.place[s].block = b;
    }
    // Pieces of at most `each` steps: the least, of sixteen lengths, with which they
    // number no more than fill the GPU once, or the last one, of which that is sure
    // unless the blocks alone are many.
    int count = 0;
    for (int b = t; b < blocks; b += 1024) count += (int)steps[b];
    int unused;
    const int total = scan1024(count, unused, wsum);
    const int fill = fill_pieces(kv.kvh), room = max(fill - blocks, (fill + 1) / 2);
    const int least = max(PR_MIN_TILES, (total + fill - 1) / fill);
    const int most = max(least, (total + room - 1) / room);
    auto length = [&](int i) { return least + (int)((long long)(most - least) * i / (TRIES - 1)); };
    int pieces = 0;
    for (int b = lane; b < blocks; b += 64) pieces += ((int)steps[b] - 1) / length(wave) + 1;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) pieces += __shfl_xor(pieces, o, 64);
    if (lane == 0) tried[wave] = pieces;
    __syncthreads();
    int each = most;
    for (int i = TRIES - 1; i >= 0; --i)
        if (tried[i] <= fill) each = length(i);
    int parts = 0;
    for (int b = 0; b < blocks; b += 1024) {
        Block blk{};
        int x = 0, k = 0, before;
        if (b + t < blocks) {
            blk = sp.blocks[b + t];
            x = (int)steps[b + t];
            k = (x - 1) / each + 1;
        }
        const int all = scan1024(k, before, wsum);
        for (int i = 0; i < k; ++i)
            sp.pieces[parts + before + i] = Piece{
                blk.row, b + t, (int)((long long)x * i / k), (int)((long long)x * (i + 1) / k),
                parts + before + i, 0, blk.toks, shares(blk.row) << kv.shift};
        if (k) sp.blocks[b + t] = Block{blk.row, blk.toks, parts + before, k};
        parts += all;
    }
    // The slots' own positions, by the few-row form: pieces of at most `length` tiles,
    // so long that they number FEW_PIECES at most (or half as many beside a piece for
    // each slot and head, where those are many).
    const int tile = kv.type == KV_T_Q8 ? 32 : 16;
    auto tiles_of = [&](const SlotRows &r, int s) {
        const int skip = shares(s) << kv.shift;
        return r.n < 1 || r.n > few ? 0 : max(1, (r.len - skip + tile - 1) / tile);
    };
    long long all = 0;
    int units = 0;
    for (int b = 0; b < n; b += 1024) {
        const int own = b + t < n ? tiles_of(slot_rows(kv, b + t), b + t) : 0;
        int before;
        all += scan1024(own, before, wsum);
        units += __syncthreads_count(own > 0);
    }
    all *= kv.kvh;
    units *= kv.kvh;
    const int spread = max(FEW_PIECES - units, FEW_PIECES / 2);
    const long long piece = max(1ll, (all + spread - 1) / spread);
    int workers = 0;
    for (int b = 0; b < n; b += 1024) {
        const int s = b + t;
        const SlotRows r = s < n ? slot_rows(kv, s) : SlotRows{};
        const int own = s < n ? tiles_of(r, s) : 0;
        const int ways = (int)((own + piece - 1) / piece);
        int before;
        const int in_all = scan1024(ways * kv.kvh, before, wsum);
        if (s < n) {
            SharedPlace p{r.begin, own ? r.n : 0, 0, 0, 0, 0, workers + before, ways};
            if (shares(s)) {
                const SharedPlace at = sp.place[s];
                const Block blk = sp.blocks[at.block];
                p.part = blk.part, p.pieces = blk.pieces, p.row = at.row, p.block = at.block;
            }
            sp.place[s] = p;
            base[s] = workers + before;
        }
        workers += in_all;
    }
    __syncthreads();
    for (int w = t; w < min(workers, sp.few_most); w += 1024) {
        int s = 0, hi = n; // the last slot with base[s] <= w
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (base[mid] <= w) s = mid;
            else hi = mid;
        }
        const SlotRows r = slot_rows(kv, s);
        const int own = tiles_of(r, s), ways = (int)((own + piece - 1) / piece);
        if (!ways) continue; // (there is none such: the last slot before w has pieces)
        const int kh = (w - base[s]) / ways, i = (w - base[s]) % ways;
        sp.few[w] = FewPiece{s,       kh,  (int)((long long)own * i / ways),
                             (int)((long long)own * (i + 1) / ways),
                             r.begin, r.n, r.len,
                             shares(s) << kv.shift, ways, {}};
    }
    if (t == 0) *sp.head = SharedHead{Plan{blocks, parts}, min(workers, sp.few_most)};
}

} // namespace

int launch_shared_plan(const PagedKv &kv, const int *group, void *plan, void *stream)
{
    const SharedPlan sp = shared_plan(plan, kv.seqs, kv.kvh, kv.heads);
    const int few = paged_few_rows(kv.heads / kv.kvh);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(shared_runs_kernel, dim3(kv.seqs), dim3(256), 0, st, kv, group, few,
                       sp.leader, sp.run);
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(1024),
                       (size_t)kv.seqs * 24 + (size_t)sp.cap * 4, st, kv, few, sp);
    return (int)hipGetLastError();
}

} // namespace hyq
