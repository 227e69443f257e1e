// What a worker of the attention over shared prefixes takes from the plan, cut to
// what there is: a plan may be of another batch, or hold any bytes. Constant
// expressions without the GPU's headers, which a host program can check as they are.
#pragma once

#include "hyq_paged.hpp"

namespace hyq {

// A range of steps of a block, with what its workgroup needs to begin.
struct Piece {
    int slot, index, t0, t1;
    int part;            // the partial block it writes, -1 for the output
    int begin, n, first; // the slot's rows, and the first one's position
};
struct SharedPlace {
    int begin, n;     // the slot's rows (n = 0: not of the few-row form)
    int part, pieces; // of its block (0 pieces: in no group); narrow: the block's first
                      // worker and its workers for each KV head
    int row;          // the slot's first row there
    int first, ways;  // its first worker, and its workers for each KV head
    int unused;
};
struct FewPiece {
    int slot, kh, t0, t1;      // tiles of the slot's positions from skip on
    int begin, n, len, skip;   // the slot's rows and positions
    int ways;                  // pieces of the slot
    int narrow;                // a block: n places of the list from begin on, len positions
    int unused[2];
};
// The sizes that a plan's numbers are cut to.
struct PlanSizes {
    int seqs, kvh, rows, stride, shift; // of the batch
    int tq, cap, most, few_most;        // a block's tokens, blocks, pieces of both forms
    constexpr long long positions() const { return (long long)stride << shift; }
};

constexpr int cut_to(int x, int least, int most)
{
    return x < least ? least : x > most ? most : x;
}
constexpr int cut_to(long long x, long long least, long long most)
{
    return (int)(x < least ? least : x > most ? most : x);
}

// A worker's piece of the few-row form, in steps of `tile` positions.
constexpr FewPiece cut_few_piece(const PlanSizes &z, int tile, FewPiece f)
{
    f.slot = cut_to(f.slot, 0, z.seqs - 1);
    f.kh = cut_to(f.kh, 0, z.kvh - 1);
    // (begin: a row there is, read whatever n)
    const int places = f.narrow ? z.cap * z.tq : z.rows;
    f.begin = cut_to(f.begin, 0, places - 1);
    f.n = cut_to(f.n, 0, places - f.begin);
    if (f.narrow && f.n > z.tq / 8) f.n = z.tq / 8;
    f.len = cut_to((long long)f.len, 0ll, z.positions());
    f.skip = cut_to(f.skip, 0, f.len) & ~15;
    const int tiles = (f.len - f.skip + tile - 1) / tile;
    f.t0 = cut_to(f.t0, 0, tiles > 0 ? tiles - 1 : 0);
    f.t1 = cut_to(f.t1, f.t0 + 1, tiles > 0 ? tiles : 1);
    return f;
}

// A workgroup's piece of the tile form. (Its steps end with the prefix, whatever t1,
// and a list's entry is looked at before it is used.)
constexpr Piece cut_piece(const PlanSizes &z, int step, Piece p)
{
    p.slot = cut_to(p.slot, 0, z.seqs - 1);
    p.index = cut_to(p.index, 0, z.cap - 1);
    p.part = cut_to(p.part, 0, z.most - 1);
    p.first = cut_to((long long)p.first, 0ll, z.positions());
    p.t0 = cut_to(p.t0, 0, p.first / step);
    p.t1 = cut_to(p.t1, 0, p.first / step + 1);
    return p;
}

// The parts that the merge joins for a slot and KV head kh: `ways` from worker
// `first` on, and `pieces` of the prefix's from `part` on, of row `row` and those
// behind it.
constexpr SharedPlace cut_place(const PlanSizes &z, int kh, bool narrow, SharedPlace p)
{
    p.begin = cut_to(p.begin, 0, z.rows);
    p.n = cut_to(p.n, 0, z.rows - p.begin);
    const int most = narrow ? z.few_most : z.most;
    p.part = cut_to(p.part, 0, most - 1);
    p.pieces = cut_to(p.pieces, 0, most - p.part);
    if (narrow)
        p.part = cut_to((long long)p.part + (long long)kh * p.pieces, 0ll,
                        (long long)most - p.pieces);
    p.ways = cut_to(p.ways, 0, z.few_most);
    p.first = cut_to((long long)(p.first > 0 ? p.first : 0) + (long long)kh * p.ways, 0ll,
                     (long long)z.few_most);
    p.ways = cut_to(p.ways, 0, z.few_most - p.first);
    return p;
}

} // namespace hyq
