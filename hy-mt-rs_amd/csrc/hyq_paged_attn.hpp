// What the two forms of the paged attention share: the slots' rows, the plan of
// the tile form (made by a workgroup of the few-row form's launch) and the
// layout of its scratch.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_paged.hpp"
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
// A range of steps of a block, with what its workgroup needs to begin.
struct Piece {
    int slot, index, t0, t1;
    int part;            // the partial block it writes, -1 for the output
    int begin, n, first; // the slot's rows, and the first one's position
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

// hyq_paged_few.hip: slots of at most `few` <= paged_few_rows(heads / kv_heads)
// new rows, with the plan where there is a tile form; and the merge of both.
int paged_few_rows(int rep);
size_t paged_few_scratch(bool f16, int seqs, int kvh, int heads, int few);
int launch_paged_few(const PagedKv &kv, int few, const RowsScratch &rs, const float *q, float *part,
                     float *out, void *stream);
int launch_paged_merge(const PagedKv &kv, int few, const RowsScratch &rs, const float *part,
                       float *out, void *stream);
// hyq_paged_rows.hip: the slots of more.
int launch_paged_rows(const PagedKv &kv, const RowsScratch &rs, const float *q, float *out,
                      void *stream);

} // namespace hyq
