// Rules on rows of logits before a token is drawn: penalties for tokens that a row
// has already, biases and grammar masks, in one pass.
//
//   l' = l / r or l * r (l > 0 or not) for a token of the row's history,
//   l' -= presence + frequency n for one that it has made n > 0 times,
//   l' += bias (of several pairs of one token the last), -inf where the mask's bit is 0.
//
// A workgroup takes CHUNK logits of a row. It holds their counts in LDS, which it
// fills from the row's whole history (a few KB, which the row's other workgroups
// read too and find in the caches): whole numbers, so that the order of the
// atomics does not matter, and of a token's biases the greatest place, not a sum.
// Nothing is sorted, and no launch waits for another. (512 and 1024 threads, which
// read the histories less often, and 4 and 16 logits a thread took as long or longer.)
//
// Two rows of 120,818 take 4.2 us, a launch. 64 rows of 128,167 with histories of up
// to 4,000 tokens, 300 biases and 8 masks take 17.5 us for 66 MB: a copy of the logits
// takes 10, 2.8 are the histories, 1.5 the masks. Longer histories bound it, which each
// of a row's 63 workgroups reads: 64 rows with 1,000 tokens each 14.5 us, 4,000 16.5,
// 16,000 33, 131,072 171. In place, where a logit is read if a rule changes it, after
// the counts are known: 12.0, 18.9, 36 and 174, and 7.4 without histories (13.2 to
// another buffer).
#include <hip/hip_runtime.h>

#include "hyq_paged.hpp"

namespace hyq {

namespace {

constexpr int THREADS = 256, PER = 8, CHUNK = THREADS * PER;
constexpr unsigned PROMPT = 0x80000000u; // a count's mark of a token that the prompt has

// KEEP: the output is the input; logits that no rule changes are not read.
template <bool KEEP>
__global__ __launch_bounds__(THREADS) void logits_adjust_kernel(const float *logits, int vocab,
                                                            LogitRulesArgs a, float *out)
{
    __shared__ unsigned count[CHUNK];
    __shared__ int pair[CHUNK]; // 1 + the last of the row's pairs for a token
    const int t = threadIdx.x, row = blockIdx.y;
    const int v0 = blockIdx.x * CHUNK, n = min(CHUNK, vocab - v0);
    const float *src = logits + (size_t)row * vocab + v0;
    float *dst = out + (size_t)row * vocab + v0;
    float x[PER];
    if constexpr (!KEEP) { // (in flight while the history is read)
#pragma unroll
        for (int k = 0; k < PER; ++k) x[k] = __builtin_nontemporal_load(src + min(t + THREADS * k, n - 1));
    }
    int held = 0, prompt = 0, from = 0, to = 0;
    if (a.history) {
        held = min(max(a.history_len[row], 0), a.history_stride);
        prompt = a.prompt_len ? a.prompt_len[row] : 0;
    }
    if (a.bias_start) {
        from = min(max(a.bias_start[row], 0), a.biases);
        to = min(max(a.bias_start[row + 1], from), a.biases);
    }
    float r = a.repetition ? a.repetition[row] : 1.f;
    r = r > 0.f ? r : 1.f;
    const float presence = a.presence ? a.presence[row] : 0.f;
    const float frequency = a.frequency ? a.frequency[row] : 0.f;
    // (a wave's 64 logits have two words of a mask, the same for all its lanes)
    const int which = a.mask ? a.mask_row[row] : -1, words = (vocab + 31) / 32;
    const unsigned *mask =
        (unsigned)which < (unsigned)a.masks ? a.mask + (size_t)which * words : nullptr;
    const int w0 = __builtin_amdgcn_readfirstlane((v0 + t) >> 5);
    unsigned long long bits[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        bits[k] = ~0ull;
        if (mask)
            bits[k] = mask[min(w0 + THREADS / 32 * k, words - 1)] |
                      (unsigned long long)mask[min(w0 + THREADS / 32 * k + 1, words - 1)] << 32;
    }
    const bool biased = to > from;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        count[t + THREADS * k] = 0;
        if (biased) pair[t + THREADS * k] = 0;
    }
    const int *history = a.history + (size_t)row * a.history_stride;
    int token[4];
    auto fetch = [&](int b) { // (four loads in flight)
#pragma unroll
        for (int k = 0; k < 4; ++k) token[k] = history[min(b + THREADS * k, held - 1)] - v0;
    };
    if (t < held) fetch(t);
    __syncthreads();
    for (int b = t; b < held; b += THREADS * 4) {
        if (b != t) fetch(b);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = b + THREADS * k;
            if (i < held && (unsigned)token[k] < (unsigned)n) {
                if (i < prompt) atomicOr(count + token[k], PROMPT);
                else atomicAdd(count + token[k], 1u);
            }
        }
    }
    for (int i = from + t; i < to; i += THREADS) {
        const int v = a.bias_token[i] - v0;
        if ((unsigned)v < (unsigned)n) atomicMax(pair + v, i + 1);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = t + THREADS * k;
        if (i >= n) break;
        const unsigned c = count[i], made = c & ~PROMPT;
        const int p = biased ? pair[i] : 0;
        const bool allowed = __builtin_amdgcn_inverse_ballot_w64(bits[k]);
        if constexpr (KEEP) {
            if (allowed && !c && !p) continue;
            x[k] = allowed ? src[i] : 0.f;
        }
        float y = x[k];
        if (c) y = y > 0.f ? y / r : y * r;
        if (made) y -= presence + frequency * (float)made;
        if (p) y += a.bias[p - 1];
        __builtin_nontemporal_store(allowed ? y : -INFINITY, dst + i);
    }
}

} // namespace

int launch_logits_adjust(const float *logits, int rows, int vocab, const LogitRulesArgs &a,
                         float *out, void *stream)
{
    const dim3 grid((vocab + CHUNK - 1) / CHUNK, rows);
    auto kernel = out == logits ? logits_adjust_kernel<true> : logits_adjust_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, (hipStream_t)stream, logits, vocab, a, out);
    return (int)hipGetLastError();
}

} // namespace hyq
