// Rules on logits before a token is chosen.  Row r counts the tokens of a list (what its request has read and said so far) and,
// of a drafted tree, those on its own path.  With c the times token v was said (the list behind its first `prompt_len` tokens, and
// the path) and s whether it was said or stood in the prompt:
//     x = s ? (x > 0 ? x / repetition : x * repetition) : x
//     x = x - frequency * c - presence * (c > 0)
//     x = x + every bias that the row gives v
//     x = -inf  where the row's grammar mask has no bit for v
// Token ids outside the vocabulary are passed over.
#include "common.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int CHUNK = 8192;                     // logits of a block: 32 KB of counts
constexpr unsigned ASKED = 0x80000000u;         // beside a count: the token stands in the prompt

struct RuleArgs {
    float* out;                    // [rows, vocab], rows `out_stride` elements apart; may be the logits themselves
    const float* logits;
    const float* penalties;        // [rows, 3]: repetition, frequency, presence
    const int* history;            // the lists' tokens, one list behind another
    const int* history_start;      // [lists + 1]
    const int* prompt_len;         // [lists]
    const int* list_of_row;        // [rows], negative: no list; null: row r has list r
    const int* drafted;            // [rows] tokens, null without trees
    const int* ancestors;          // [rows, words]: bits of the nodes on the row's path, itself among them
    const int* first_row;          // [rows]: the row of the first node of its tree
    const int* bias_start;         // [rows + 1], null without biases
    const int* bias_tokens;
    const float* bias_values;
    const int* mask;               // [masks, mask_words], bit v: token v may follow; null without masks
    const int* mask_of_row;        // [rows], negative: no mask; null: row r has mask r
    long long out_stride, in_stride, history_len, bias_len;
    int rows, lists, vocab, words, masks, mask_words;
};

__device__ __forceinline__ float ruled(float x, unsigned count, float rep, float freq, float pres) {
    if (count == 0u) return x;
    x = x > 0.f ? x / rep : x * rep;
    const unsigned c = count & ~ASKED;
    if (c) x = x - freq * (float)c - pres;
    return x;
}

__global__ void __launch_bounds__(THREADS)
logit_rules_kernel(const RuleArgs A) {
    __shared__ unsigned count[CHUNK];
    const int r = blockIdx.y, lo = (int)blockIdx.x * CHUNK, n = min(CHUNK, A.vocab - lo);
    const int list = A.list_of_row ? A.list_of_row[r] : r;
    for (int i = threadIdx.x; i < n; i += THREADS) count[i] = 0u;
    __syncthreads();
    if (list >= 0 && list < A.lists) {
        const long long a = max(0, A.history_start[list]), z = min((long long)A.history_start[list + 1], A.history_len);
        const long long said = a + A.prompt_len[list];
        for (long long i = a + threadIdx.x; i < z; i += THREADS) {
            const unsigned u = (unsigned)(A.history[i] - lo);
            if (u < (unsigned)n) {
                if (i < said) atomicOr(&count[u], ASKED);
                else atomicAdd(&count[u], 1u);
            }
        }
    }
    if (A.drafted) {
        const long long first = A.first_row[r];
        for (int i = threadIdx.x; i < A.words * 32; i += THREADS) {
            if (!(A.ancestors[(size_t)r * A.words + (i >> 5)] >> (i & 31) & 1)) continue;
            if (first + i < 0 || first + i >= A.rows) continue;
            const unsigned u = (unsigned)(A.drafted[first + i] - lo);
            if (u < (unsigned)n) atomicAdd(&count[u], 1u);
        }
    }
    __syncthreads();
    const float rep = A.penalties[3 * r], freq = A.penalties[3 * r + 1], pres = A.penalties[3 * r + 2];
    const int m = A.mask == nullptr ? -1 : (A.mask_of_row ? A.mask_of_row[r] : r);
    const int* mask = m >= 0 && m < A.masks ? A.mask + (size_t)m * A.mask_words : nullptr;
    const float* in = A.logits + (size_t)r * A.in_stride + lo;
    float* out = A.out + (size_t)r * A.out_stride + lo;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const bool may = mask == nullptr || (mask[(lo + i) >> 5] >> ((lo + i) & 31) & 1);
        out[i] = may ? ruled(in[i], count[i], rep, freq, pres) : -INFINITY;
    }
    if (!A.bias_start) return;
    __syncthreads();
    // a token that several entries name gets their sum, in their order, from the thread of the first
    const long long a = max(0, A.bias_start[r]), z = min((long long)A.bias_start[r + 1], A.bias_len);
    for (long long i = a + threadIdx.x; i < z; i += THREADS) {
        const int v = A.bias_tokens[i];
        const unsigned u = (unsigned)(v - lo);
        if (u >= (unsigned)n) continue;
        if (mask != nullptr && !(mask[v >> 5] >> (v & 31) & 1)) continue;
        bool first = true;
        for (long long j = a; j < i && first; ++j) first = A.bias_tokens[j] != v;
        if (!first) continue;
        float x = out[u];
        for (long long j = i; j < z; ++j)
            if (A.bias_tokens[j] == v) x += A.bias_values[j];
        out[u] = x;
    }
}

}  // namespace

XB_EXPORT int xb_logit_rules(float* out, const float* logits, const float* penalties, const int* history, const int* history_start, const int* prompt_len,
                             const int* list_of_row, const int* drafted, const int* ancestors, const int* first_row, const int* bias_start,
                             const int* bias_tokens, const float* bias_values, const int* mask, const int* mask_of_row, long long out_stride,
                             long long in_stride, long long history_len, long long bias_len, int rows, int lists, int vocab, int words, int masks,
                             int mask_words, cudaStream_t stream) {
    if (rows <= 0 || vocab <= 0) return 0;
    if (rows > 65535 || (mask && mask_words < (vocab + 31) / 32)) return (int)cudaErrorInvalidValue;
    const RuleArgs A{out, logits, penalties, history, history_start, prompt_len, list_of_row, drafted, ancestors, first_row, bias_start, bias_tokens,
                     bias_values, mask, mask_of_row, out_stride, in_stride, history_len, bias_len, rows, lists, vocab, words, masks, mask_words};
    logit_rules_kernel<<<dim3((vocab + CHUNK - 1) / CHUNK, rows), THREADS, 0, stream>>>(A);
    return xb_launch_status();
}
