// Bookkeeping of a paged KV cache on the device: forking, trimming and freeing
// slots, giving slots the pages of their next tokens, and moving the live
// pages to the front of the pool. Tables, lengths and counts stay in device
// memory and every result is exact and independent of the order in which
// threads run (integer counts; the lowest free page first; slots in order),
// so a whole serving step can be enqueued, or captured in a graph, without
// the host.
//
// Where nothing is copied these are launches and dependent loads: a fork and an
// extension of 8 slots take 10 to 13 us, of 128 slots over 20,000 to 200,000 pages
// 33 (the larger forms below). A compaction's plan, by one workgroup, grows with
// the pool: 8 us for 700 pages, 53 for 20,000, 460 for 200,000. Copies are bound by memory: 128 beams of
// 32 layers, 4 heads, f16, whose last pages are copied 42 us in all (the copies
// 31, of rows scattered over a pool of 10 GB), a compaction that reads and writes
// 1.3 GB 253 us (5.2 TB/s, what a copy reaches). 8-bit pages take about half: the copies
// of 128 beams' last pages 46 us where f16 ones take 98, a compaction's moves 123 and 248.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged.hpp"

namespace hyq {

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int held_pages(int len, int shift, int stride)
{
    return min((int)(((long long)max(len, 0) + (1 << shift) - 1) >> shift), stride);
}

// ---- fork ----
// table_out[s] = the entries that hold the first min(len[p], keep[s])
// positions of slot p = parent[s] (none for a p outside the table).
// Grid: one workgroup per slot, then workgroups that clear the counts.
__global__ __launch_bounds__(256) void pages_fork_kernel(PagesArgs a, const int *__restrict__ parent,
                                                         const int *__restrict__ keep,
                                                         const int *__restrict__ table,
                                                         const int *__restrict__ len,
                                                         int *__restrict__ table_out,
                                                         int *__restrict__ len_out,
                                                         int *__restrict__ refs_out)
{
    const int t = threadIdx.x;
    if ((int)blockIdx.x >= a.seqs) {
        const int n = (gridDim.x - a.seqs) * 256;
        for (int i = (blockIdx.x - a.seqs) * 256 + t; i < a.npages; i += n) refs_out[i] = 0;
        return;
    }
    const int s = blockIdx.x, p = parent[s];
    int got = 0;
    if ((unsigned)p < (unsigned)a.seqs) {
        got = (int)min((long long)max(len[p], 0), (long long)a.stride << a.shift);
        if (keep) got = min(got, max(keep[s], 0));
    }
    const int n = held_pages(got, a.shift, a.stride);
    const int *src = table + (size_t)(n ? p : 0) * a.stride;
    int *dst = table_out + (size_t)s * a.stride;
    for (int i = t; i < a.stride; i += 256) dst[i] = i < n ? src[i] : -1;
    if (t == 0) len_out[s] = got;
}

// refs[p] = the entries that name page p, over the entries in use.
__global__ __launch_bounds__(256) void pages_count_kernel(PagesArgs a, const int *__restrict__ table,
                                                          const int *__restrict__ len,
                                                          int *__restrict__ refs)
{
    const int s = blockIdx.x;
    const int n = held_pages(len[s], a.shift, a.stride);
    for (int i = threadIdx.x; i < n; i += 256) {
        const int p = table[(size_t)s * a.stride + i];
        if ((unsigned)p < (unsigned)a.npages) atomicAdd(refs + p, 1);
    }
}

// Both by one workgroup, the counts in LDS, where table and pool are small: one
// launch instead of two. (With the small form of the extension, against the two
// larger ones in the same small pool: 8 slots 12 and 28 us a step, 128 slots, with
// copies that took longer then, 54 and 73.)
constexpr int SMALL_PAGES = 4096, SMALL_SLOTS = 1024, SMALL_ENTRIES = 16384;
__global__ __launch_bounds__(1024) void pages_fork_small_kernel(
    PagesArgs a, const int *__restrict__ parent, const int *__restrict__ keep,
    const int *__restrict__ table, const int *__restrict__ len, int *__restrict__ table_out,
    int *__restrict__ len_out, int *__restrict__ refs_out)
{
    extern __shared__ int count[]; // [npages]
    __shared__ int from[SMALL_SLOTS], used[SMALL_SLOTS];
    const int t = threadIdx.x;
    for (int i = t; i < a.npages; i += 1024) count[i] = 0;
    if (t < a.seqs) {
        const int p = parent[t];
        int got = 0;
        if ((unsigned)p < (unsigned)a.seqs) {
            got = (int)min((long long)max(len[p], 0), (long long)a.stride << a.shift);
            if (keep) got = min(got, max(keep[t], 0));
        }
        len_out[t] = got;
        from[t] = p;
        used[t] = held_pages(got, a.shift, a.stride);
    }
    __syncthreads();
    const int n = a.seqs * a.stride;
    for (int i = t; i < n; i += 1024) {
        const int s = i / a.stride, e = i - s * a.stride;
        int p = -1;
        if (e < used[s]) {
            p = table[from[s] * a.stride + e];
            if ((unsigned)p < (unsigned)a.npages) atomicAdd(count + p, 1);
        }
        table_out[i] = p;
    }
    __syncthreads();
    for (int i = t; i < a.npages; i += 1024) refs_out[i] = count[i];
}

// ---- extend ----
// Scratch of the plans, in ints.
struct PagesScratch {
    int *count;  // [16]: copies / moves, live pages
    int *top;    // [npages]
    int *asks;   // [npages]
    int *free;   // [npages]
    int *need;   // [seqs]: 2 * pages a slot wants + whether it copies
    int *list;   // [3 max(npages, seqs)]
};
__device__ inline PagesScratch pages_layout(void *scratch, int npages, int seqs)
{
    PagesScratch p;
    p.count = (int *)scratch;
    p.top = p.count + 16;
    p.asks = p.top + npages;
    p.free = p.asks + npages;
    p.need = p.free + npages;
    p.list = p.need + seqs;
    return p;
}

__device__ __forceinline__ int fresh(const int *p) // past this workgroup's own cached line
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive scan over 1024 threads; returns the total.
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

struct Ask {
    int held, wants, fill, last;
    bool asks, is_long, partial;
};
__device__ __forceinline__ Ask ask_of(const PagesArgs &a, const int *add, const int *table,
                                      const int *len, int s)
{
    Ask k;
    const int n = max(len[s], 0), more = add[s];
    const long long cap = (long long)a.stride << a.shift;
    k.is_long = more > 0 && (long long)n + more > cap;
    k.asks = more > 0 && !k.is_long;
    k.held = held_pages(n, a.shift, a.stride);
    k.wants = k.asks ? held_pages(n + more, a.shift, a.stride) : k.held;
    k.fill = n & ((1 << a.shift) - 1);
    k.last = k.held > 0 ? table[(size_t)s * a.stride + k.held - 1] : -1;
    k.partial = k.asks && k.fill > 0 && (unsigned)k.last < (unsigned)a.npages;
    return k;
}

// The tables and counts that the plan writes elsewhere, by many workgroups.
__global__ __launch_bounds__(256) void pages_copy_kernel(const int *__restrict__ table,
                                                         int *__restrict__ table_out,
                                                         size_t entries,
                                                         const int *__restrict__ refs,
                                                         int *__restrict__ refs_out, int npages)
{
    const size_t first = (size_t)blockIdx.x * 256 + threadIdx.x, step = (size_t)gridDim.x * 256;
    for (size_t i = first; i < entries; i += step) table_out[i] = table[i];
    for (size_t i = first; i < (size_t)npages; i += step) refs_out[i] = refs[i];
}

// One workgroup of 1024 threads. A slot's partly filled last page that others
// name too is copied for it, unless all who name the page extend it in this
// call and the slot holds most of it (the first of those): that one goes on
// writing behind what any other has. Slots are served in order while free
// pages last.
__global__ __launch_bounds__(1024) void pages_extend_kernel(
    PagesArgs a, const int *__restrict__ add, const int *table, const int *len, const int *refs,
    int *table_out, int *len_out, int *refs_out, int *__restrict__ status,
    int *__restrict__ served_len, void *scratch)
{
    __shared__ int wsum[16];
    const PagesScratch w = pages_layout(scratch, a.npages, a.seqs);
    const int t = threadIdx.x;
    for (int s = t; s < a.seqs; s += 1024) {
        const Ask k = ask_of(a, add, table, len, s);
        if (k.partial && refs[k.last] > 1) {
            w.top[k.last] = 0;
            w.asks[k.last] = 0;
        }
    }
    __threadfence();
    __syncthreads();
    for (int s = t; s < a.seqs; s += 1024) {
        const Ask k = ask_of(a, add, table, len, s);
        if (k.partial && refs[k.last] > 1) {
            atomicAdd(w.asks + k.last, 1);
            atomicMax((unsigned *)w.top + k.last, (unsigned)k.fill << 16 | (65535u - s));
        }
    }
    __threadfence();
    __syncthreads();
    auto copies_of = [&](const Ask &k, int s) {
        if (!k.partial || refs[k.last] <= 1) return false;
        const bool keeps = fresh(w.asks + k.last) == refs[k.last] &&
                           (unsigned)fresh(w.top + k.last) ==
                               ((unsigned)k.fill << 16 | (65535u - s));
        return !keeps;
    };
    // how many pages all slots want, and as many free ones, lowest first
    int total = 0;
    for (int b = 0; b < a.seqs; b += 1024) {
        int need = 0, before;
        if (b + t < a.seqs) {
            const Ask k = ask_of(a, add, table, len, b + t);
            const bool copies = copies_of(k, b + t);
            if (k.asks) need = k.wants - k.held + copies;
            w.need[b + t] = 2 * need + copies;
        }
        total += scan1024(need, before, wsum);
        total = min(total, a.npages + 1); // (no more than that matters)
    }
    int found = 0;
    for (int b = 0; b < a.npages && found < total; b += 1024) {
        const int p = b + t;
        const int is = p < a.npages && refs[p] == 0;
        int before;
        const int all = scan1024(is, before, wsum);
        if (is && found + before < total) w.free[found + before] = p;
        found += all;
    }
    // (the counts in `refs` are not read again: where refs_out is refs they change
    // now, elsewhere the launch before has copied them, and the table)
    __threadfence();
    __syncthreads();
    int carry = 0, ncopies = 0;
    for (int b = 0; b < a.seqs; b += 1024) {
        const int s = b + t;
        Ask k{};
        bool copies = false;
        int need = 0, before, cbefore;
        if (s < a.seqs) {
            k = ask_of(a, add, table, len, s);
            copies = w.need[s] & 1;
            need = w.need[s] >> 1;
        }
        const int all = scan1024(need, before, wsum);
        const long long upto = (long long)carry + before + need;
        const bool served = k.asks && (need == 0 || upto <= found);
        const int call = scan1024(served && copies, cbefore, wsum);
        if (s < a.seqs) {
            int n = max(len[s], 0);
            if (served) {
                int at = carry + before;
                int *row = table_out + (size_t)s * a.stride;
                if (copies) {
                    const int p = w.free[at++];
                    row[k.held - 1] = p;
                    __hip_atomic_store(refs_out + p, 1, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
                    atomicSub(refs_out + k.last, 1);
                    int *c = w.list + 3 * (ncopies + cbefore);
                    c[0] = k.last;
                    c[1] = p;
                    c[2] = k.fill;
                }
                for (int i = k.held; i < k.wants; ++i) {
                    const int p = w.free[at++];
                    row[i] = p;
                    __hip_atomic_store(refs_out + p, 1, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
                }
                n += add[s];
            }
            len_out[s] = n;
            const int refused = k.is_long ? 2 : k.asks && !served ? 1 : 0;
            status[s] = refused;
            if (served_len) served_len[s] = refused ? 0 : n;
        }
        carry = min(carry + all, a.npages + 1);
        ncopies += call;
        __syncthreads();
    }
    if (t == 0) w.count[0] = ncopies;
}

// The same for at most SMALL_SLOTS slots and SMALL_PAGES pages, a slot and four
// pages per thread, with the counts in LDS: what the larger form does in rounds
// of global memory takes a load, a dependent load and a few barriers (21 -> 8 us
// for 8 slots and 260 pages).
__global__ __launch_bounds__(1024) void pages_extend_small_kernel(
    PagesArgs a, const int *__restrict__ add, const int *table, const int *len, const int *refs,
    int *table_out, int *len_out, int *refs_out, int *__restrict__ status,
    int *__restrict__ served_len, void *scratch, int copy)
{
    extern __shared__ int lds[];
    __shared__ int wsum[16];
    const PagesScratch w = pages_layout(scratch, a.npages, a.seqs);
    int *const lrefs = lds, *const asks = lrefs + a.npages;
    unsigned *const top = (unsigned *)(asks + a.npages);
    int *const free = asks; // (once the asks are counted)
    const int t = threadIdx.x, s = t;
    constexpr int EACH = SMALL_PAGES / 1024;
    int r[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) r[i] = refs[min(EACH * t + i, a.npages - 1)];
    Ask k{};
    int n = 0;
    if (s < a.seqs) {
        k = ask_of(a, add, table, len, s);
        n = max(len[s], 0);
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (EACH * t + i < a.npages) {
            lrefs[EACH * t + i] = r[i];
            asks[EACH * t + i] = 0;
            top[EACH * t + i] = 0;
        }
    if (copy)
        for (int i = t; i < a.seqs * a.stride; i += 1024) table_out[i] = table[i];
    __syncthreads();
    const bool shared = k.partial && lrefs[k.last] > 1;
    const unsigned key = (unsigned)k.fill << 16 | (65535u - s);
    if (shared) {
        atomicAdd(asks + k.last, 1);
        atomicMax(top + k.last, key);
    }
    __syncthreads();
    const bool copies = shared && !(asks[k.last] == lrefs[k.last] && top[k.last] == key);
    const int need = k.asks ? k.wants - k.held + copies : 0;
    int before, fbefore, cbefore, is = 0;
    const int total = scan1024(need, before, wsum);
#pragma unroll
    for (int i = 0; i < EACH; ++i) is += EACH * t + i < a.npages && r[i] == 0;
    const int found = scan1024(is, fbefore, wsum);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (EACH * t + i < a.npages && r[i] == 0 && fbefore < total) free[fbefore++] = EACH * t + i;
    const bool served = k.asks && (need == 0 || before + need <= found);
    const int ncopies = scan1024(served && copies, cbefore, wsum); // (and the list is whole)
    if (s < a.seqs) {
        if (served) {
            int at = before;
            int *row = table_out + (size_t)s * a.stride;
            if (copies) {
                const int p = free[at++];
                row[k.held - 1] = p;
                lrefs[p] = 1;
                atomicSub(lrefs + k.last, 1);
                int *c = w.list + 3 * cbefore;
                c[0] = k.last;
                c[1] = p;
                c[2] = k.fill;
            }
            for (int i = k.held; i < k.wants; ++i) {
                const int p = free[at++];
                row[i] = p;
                lrefs[p] = 1;
            }
            n += add[s];
        }
        len_out[s] = n;
        const int refused = k.is_long ? 2 : k.asks && !served ? 1 : 0;
        status[s] = refused;
        if (served_len) served_len[s] = refused ? 0 : n;
    }
    if (t == 0) w.count[0] = ncopies;
    __syncthreads();
    for (int i = t; i < a.npages; i += 1024) refs_out[i] = lrefs[i];
}

// Copies the filled rows of the pages on the list: one wave per (page, layer,
// keys or values, head), rows of contiguous 16-byte words. Stored past the
// caches: 128 beams' step 54 -> 43 us.
__global__ __launch_bounds__(256) void pages_fill_kernel(PagesArgs a, char *pool, void *scratch)
{
    const PagesScratch w = pages_layout(scratch, a.npages, a.seqs);
    const int n = w.count[0], per = a.layers * 2 * a.kvh;
    const int lane = threadIdx.x & 63;
    const size_t scales = a.type == KV_T_Q8 ? 4 : 0, row = kv_row_bytes(a.type) - scales;
    const size_t head = row << a.shift, page = (head + (scales << a.shift)) * 2 * a.kvh;
    const long long items = (long long)n * per, step = (long long)gridDim.x * 4;
    for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < items; i += step) {
        const int c = (int)(i / per), r = (int)(i % per);
        const int *e = w.list + 3 * c;
        const size_t at = (size_t)(r / (2 * a.kvh)) * a.npages * page + (size_t)(r % (2 * a.kvh)) * head;
        const u32x4 *src = reinterpret_cast<const u32x4 *>(pool + at + e[0] * page);
        u32x4 *dst = reinterpret_cast<u32x4 *>(pool + at + e[1] * page);
        const int words = (int)(e[2] * row / 16);
        // (eight loads in flight, those past the end of the last word again)
        for (int x = lane; x < words; x += 512) {
            u32x4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = src[min(x + 64 * k, words - 1)];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (x + 64 * k < words) __builtin_nontemporal_store(v[k], dst + x + 64 * k);
        }
        if (scales) { // (at most 256 of them, behind all heads' codes; the last words of four whole)
            const size_t by = (size_t)(r / (2 * a.kvh)) * a.npages * page + head * 2 * a.kvh +
                              (size_t)(r % (2 * a.kvh)) * (scales << a.shift) + lane * 16;
            if (lane < (e[2] + 3) / 4)
                *reinterpret_cast<u32x4 *>(pool + by + e[1] * page) =
                    *reinterpret_cast<const u32x4 *>(pool + by + e[0] * page);
        }
    }
}

// ---- compact ----
// One workgroup of 1024 threads: the live pages behind the live count, in
// order, go to the free ids below it, in order; `top` maps an id to its new
// one.
__global__ __launch_bounds__(1024) void pages_compact_kernel(PagesArgs a, const int *refs,
                                                             int *refs_out, int *live,
                                                             void *scratch)
{
    __shared__ int wsum[16];
    const PagesScratch w = pages_layout(scratch, a.npages, a.seqs);
    const int t = threadIdx.x;
    int count = 0;
    for (int b = 0; b < a.npages; b += 1024) {
        int before;
        count += scan1024(b + t < a.npages && refs[b + t] > 0, before, wsum);
    }
    int moves = 0, holes = 0;
    for (int b = 0; b < a.npages; b += 1024) {
        const int p = b + t;
        const bool in = p < a.npages, is = in && refs[p] > 0;
        int mb, hb;
        const int m = scan1024(is && p >= count, mb, wsum);
        const int h = scan1024(in && !is && p < count, hb, wsum);
        if (is && p >= count) w.list[moves + mb] = p;
        if (in && !is && p < count) w.free[holes + hb] = p;
        if (in) w.top[p] = p;
        moves += m;
        holes += h;
    }
    __threadfence();
    __syncthreads();
    if (refs_out != refs)
        for (int i = t; i < a.npages; i += 1024) refs_out[i] = max(refs[i], 0);
    __syncthreads();
    for (int i = t; i < moves; i += 1024) { // (holes == moves)
        const int src = fresh(w.list + i), dst = fresh(w.free + i);
        w.top[src] = dst;
        refs_out[dst] = refs[src];
        refs_out[src] = 0;
    }
    if (t == 0) {
        w.count[0] = moves;
        *live = count;
    }
}

// Moves the pages (in pieces of COMPACT_BYTES, a workgroup each) and renames
// the table's entries. 1024 workgroups: 252 us where 512 and 2048 took 259; loads
// that stay in the caches 262.
constexpr int COMPACT_BYTES = 16384;
__global__ __launch_bounds__(256) void pages_move_kernel(PagesArgs a, char *pool, const int *table,
                                                         int *table_out, void *scratch)
{
    const PagesScratch w = pages_layout(scratch, a.npages, a.seqs);
    const int t = threadIdx.x;
    const size_t page = ((size_t)kv_row_bytes(a.type) << a.shift) * 2 * a.kvh;
    const int cuts = (int)((page + COMPACT_BYTES - 1) / COMPACT_BYTES);
    const long long per = (long long)a.layers * cuts, items = w.count[0] * per;
    for (long long i = blockIdx.x; i < items; i += gridDim.x) {
        const int m = (int)(i / per), r = (int)(i % per), cut = r % cuts;
        const size_t layer = (size_t)(r / cuts) * a.npages * page + (size_t)cut * COMPACT_BYTES;
        const u32x4 *src = reinterpret_cast<const u32x4 *>(pool + layer + w.list[m] * page);
        u32x4 *dst = reinterpret_cast<u32x4 *>(pool + layer + w.free[m] * page);
        const int words = (int)min((size_t)COMPACT_BYTES, page - (size_t)cut * COMPACT_BYTES) / 16;
        u32x4 v[COMPACT_BYTES / 4096];
#pragma unroll
        for (int k = 0; k < COMPACT_BYTES / 4096; ++k)
            v[k] = __builtin_nontemporal_load(src + min(t + 256 * k, words - 1));
#pragma unroll
        for (int k = 0; k < COMPACT_BYTES / 4096; ++k)
            if (t + 256 * k < words) __builtin_nontemporal_store(v[k], dst + t + 256 * k);
    }
    const size_t n = (size_t)a.seqs * a.stride;
    for (size_t i = (size_t)blockIdx.x * 256 + t; i < n; i += (size_t)gridDim.x * 256) {
        const int p = table[i];
        table_out[i] = (unsigned)p < (unsigned)a.npages ? w.top[p] : p;
    }
}

} // namespace

size_t pages_scratch(int npages, int seqs)
{
    return (16 + 3 * (size_t)npages + seqs + 3 * (size_t)std::max(npages, seqs)) * 4;
}

int launch_pages_fork(const PagesArgs &a, const int *parent, const int *keep, const int *table,
                      const int *len, int *table_out, int *len_out, int *refs_out, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    if (a.npages <= SMALL_PAGES && a.seqs <= SMALL_SLOTS && a.seqs * a.stride <= SMALL_ENTRIES) {
        hipLaunchKernelGGL(pages_fork_small_kernel, dim3(1), dim3(1024), (size_t)a.npages * 4, st,
                           a, parent, keep, table, len, table_out, len_out, refs_out);
        return (int)hipGetLastError();
    }
    const int clears = std::min(64, (a.npages + 255) / 256);
    hipLaunchKernelGGL(pages_fork_kernel, dim3(a.seqs + clears), dim3(256), 0, st, a, parent, keep,
                       table, len, table_out, len_out, refs_out);
    hipLaunchKernelGGL(pages_count_kernel, dim3(a.seqs), dim3(256), 0, st, a, table_out, len_out,
                       refs_out);
    return (int)hipGetLastError();
}

int launch_pages_extend(const PagesArgs &a, void *pool, const int *add, const int *table,
                        const int *len, const int *refs, int *table_out, int *len_out,
                        int *refs_out, int *status, int *served, void *scratch, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    // A table that goes elsewhere is copied by the one workgroup while it is small,
    // by a launch of its own beyond (16384 entries 9.0 and 9.2 us, 32768 11.1 and
    // 9.8, 2^20 293 and 10.9; 128 slots of 512 entries over 50,000 pages, with their
    // counts, 36.6 and 19.2).
    const size_t entries = (size_t)a.seqs * a.stride;
    const bool small = a.npages <= SMALL_PAGES && a.seqs <= SMALL_SLOTS;
    const bool copy = small && table_out != table && entries <= SMALL_ENTRIES;
    const size_t nt = table_out != table && !copy ? entries : 0;
    const int nr = refs_out != refs && !small ? a.npages : 0;
    if (nt || nr) {
        const size_t groups = (std::max(nt, (size_t)nr) + 255) / 256;
        hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)std::min(groups, (size_t)1024)),
                           dim3(256), 0, st, table, table_out, nt, refs, refs_out, nr);
    }
    if (small)
        hipLaunchKernelGGL(pages_extend_small_kernel, dim3(1), dim3(1024), (size_t)a.npages * 12,
                           st, a, add, table, len, refs, table_out, len_out, refs_out, status,
                           served, scratch, (int)copy);
    else
        hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(1024), 0, st, a, add, table, len,
                           refs, table_out, len_out, refs_out, status, served, scratch);
    hipLaunchKernelGGL(pages_fill_kernel, dim3(512), dim3(256), 0, st, a, (char *)pool, scratch);
    return (int)hipGetLastError();
}

int launch_pages_compact(const PagesArgs &a, void *pool, const int *table, const int *refs,
                         int *table_out, int *refs_out, int *live, void *scratch, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(1024), 0, st, a, refs, refs_out, live,
                       scratch);
    hipLaunchKernelGGL(pages_move_kernel, dim3(1024), dim3(256), 0, st, a, (char *)pool, table,
                       table_out, scratch);
    return (int)hipGetLastError();
}

} // namespace hyq
