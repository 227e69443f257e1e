// Launchers of the paged KV cache's operators and of the sampler (kernels in
// hyq_paged_append.hip, hyq_paged_few.hip, hyq_paged_rows.hip, hyq_pages.hip
// and hyq_sample.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace hyq {

constexpr int KV_D = 128;           // head dimension
constexpr int KV_MAX_SEQS = 4096;   // slots of a page table
constexpr int KV_MAX_REP = 16;      // query heads per KV head

// One layer's pages as the kernels read them: page p holds keys
// [kv_heads][page_tokens][128] and then values of the same shape.
struct PagedKv {
    const void *pages;  // the layer's first page
    const int *table;   // [seqs][stride] page ids, -1 where none
    const int *len;     // [seqs] positions held, the new rows' among them
    const int *start;   // [seqs + 1] first new row of a slot
    int f16;            // element type: 0 f32, 1 f16
    int seqs, stride, npages, shift; // page_tokens == 1 << shift
    int kvh, heads, rows;
};

int launch_paged_append(const PagedKv &kv, const float *q, const float *k, const float *v,
                        const float *qn, const float *kn, const float *freq, float eps,
                        bool norm_first, float *q_out, void *stream);

// Attention: the one-wave form for slots of few new rows and the tile form for
// the others; scratch as paged_attention_scratch says.
size_t paged_attention_scratch(bool f16, int seqs, int kvh, int heads, int rows, int max_rows);
int launch_paged_attention(const PagedKv &kv, int max_rows, const float *q, void *scratch,
                           float *out, void *stream);

struct PagesArgs {
    int f16, layers, kvh, shift, npages, seqs, stride;
};
size_t pages_scratch(int npages, int seqs);
int launch_pages_fork(const PagesArgs &a, const int *parent, const int *keep, const int *table,
                      const int *len, int *table_out, int *len_out, int *refs_out, void *stream);
// (served: the lengths of the slots that were served, 0 for the others, or null)
int launch_pages_extend(const PagesArgs &a, void *pool, const int *add, const int *table,
                        const int *len, const int *refs, int *table_out, int *len_out,
                        int *refs_out, int *status, int *served, void *scratch, void *stream);
int launch_pages_compact(const PagesArgs &a, void *pool, const int *table, const int *refs,
                         int *table_out, int *refs_out, int *live, void *scratch, void *stream);

size_t sample_scratch(int rows, int vocab);
int launch_sample(const float *logits, int rows, int vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *random,
                  void *scratch, int *token, float *prob, void *stream);

} // namespace hyq
