// Launchers of the paged KV cache's operators and of the sampler (kernels in
// hyq_paged_*.hip, hyq_pages.hip, hyq_logits.hip and hyq_sample.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace hyq {

constexpr int KV_D = 128;           // head dimension
constexpr int KV_MAX_SEQS = 4096;   // slots of a page table
constexpr int KV_MAX_REP = 16;      // query heads per KV head

// Element types of a pool. KV_T_Q8: a byte for each number and an f32 scale for
// the 128 of a position and head, x = scale * code with codes from -127 to 127;
// a key's code as a signed byte (an operand of the int8 matrix instructions as
// it is), a value's as code + 128 (which one fma on f16 pairs turns into a code).
enum { KV_T_F32 = 0, KV_T_F16 = 1, KV_T_Q8 = 2 };
// Bytes of one position of a head.
constexpr int kv_row_bytes(int type)
{
    return type == KV_T_Q8 ? KV_D + 4 : type == KV_T_F16 ? KV_D * 2 : KV_D * 4;
}

// One layer's pages as the kernels read them: page p holds keys
// [kv_heads][page_tokens][128] and then values of the same shape; with KV_T_Q8
// behind them the scales [2][kv_heads][page_tokens].
struct PagedKv {
    const void *pages;  // the layer's first page
    const int *table;   // [seqs][stride] page ids, -1 where none
    const int *len;     // [seqs] positions held, the new rows' among them
    const int *start;   // [seqs + 1] first new row of a slot
    int type;           // KV_T_*
    int seqs, stride, npages, shift; // page_tokens == 1 << shift
    int kvh, heads, rows;
};

int launch_paged_append(const PagedKv &kv, const float *q, const float *k, const float *v,
                        const float *qn, const float *kn, const float *freq, float eps,
                        bool norm_first, float *q_out, void *stream);
// The packed rows' keys and values as f32 rows (kv.heads is not read).
int launch_paged_read(const PagedKv &kv, float *k, float *v, void *stream);

// Attention: the one-wave form for slots of few new rows and the tile form for
// the others; scratch as paged_attention_scratch says.
size_t paged_attention_scratch(int type, bool shared, int seqs, int kvh, int heads, int rows,
                               int max_rows);
// plan: of the prefixes that slots share (launch_shared_plan's), or null; their
// parts lie in the scratch behind what paged_attention_scratch says.
int launch_paged_attention(const PagedKv &kv, int max_rows, const float *q, void *scratch,
                           const void *plan, float *out, void *stream);

// The plan of a step's shared prefixes. group: the slots' groups, or null.
size_t shared_plan_bytes(int seqs, int kvh, int heads);
size_t shared_attention_scratch(int type, int seqs, int kvh, int heads, int rows, int max_rows);
// least: positions times KV heads that it is to save.
int launch_shared_plan(const PagedKv &kv, const int *group, long long least, void *plan,
                       void *stream);

struct PagesArgs {
    int type, layers, kvh, shift, npages, seqs, stride;
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

// Rules on rows of logits (hyq_logit_rules, hyq_logits.hip).
struct LogitRulesArgs {
    const int *history, *history_len, *prompt_len;
    const float *repetition, *presence, *frequency;
    const int *bias_start, *bias_token;
    const float *bias;
    const unsigned *mask;
    const int *mask_row;
    int history_stride, biases, masks;
};
int launch_logits_adjust(const float *logits, int rows, int vocab, const LogitRulesArgs &a,
                         float *out, void *stream);

size_t sample_scratch(int rows, int vocab);
int launch_sample(const float *logits, int rows, int vocab, const float *temperature,
                  const int *top_k, const float *top_p, const float *min_p, const float *random,
                  void *scratch, int *token, float *prob, void *stream);

} // namespace hyq
