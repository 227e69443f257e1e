// What the two forms of the paged attention share.
#pragma once

#include <hip/hip_runtime.h>

#include "hyq_paged.hpp"

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

// hyq_paged_few.hip: slots of at most `few` <= paged_few_rows(heads / kv_heads)
// new rows.
int paged_few_rows(int rep);
size_t paged_few_scratch(int seqs, int kvh, int heads, int few);
int launch_paged_few(const PagedKv &kv, int few, const float *q, float *part, float *out,
                     void *stream);
// hyq_paged_rows.hip: the slots of more.
size_t paged_rows_scratch(int seqs, int kvh, int heads, int rows);
int launch_paged_rows(const PagedKv &kv, const float *q, void *scratch, float *out, void *stream);

} // namespace hyq
