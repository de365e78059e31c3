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

constexpr int THREADS = 256;
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
    int rows, lists, vocab, words, masks, mask_words, rows_per_block;
};

__device__ __forceinline__ float ruled(float x, unsigned count, float rep, float freq, float pres) {
    if (count == 0u) return x;
    x = x > 0.f ? x / rep : x * rep;
    const unsigned c = count & ~ASKED;
    if (c) x = x - freq * (float)c - pres;
    return x;
}

constexpr int ROWS = 16;                        // rows of a block at most: what they need to know lies in shared memory
constexpr int WORDS = 32;                       // words of ancestors: trees of up to 1,024 nodes

struct RowFacts {
    float rep, freq, pres;
    int list, mask, first, bias, biases;
};

// A block takes 1,024 VECS tokens of the vocabulary of several rows in turn.  The lists' tokens are counted in shared memory, once for
// rows that follow each other with one list (the nodes of a tree); a row's own path is added before it and taken away behind it.  The
// next row's logits and mask are on their way meanwhile.  Bound by memory: a logit is read and written once.
template <int VECS>
__global__ void __launch_bounds__(THREADS, 4)
logit_rules_kernel(const RuleArgs A) {
    constexpr int CHUNK = 4 * THREADS * VECS;
    __shared__ __align__(16) unsigned count[CHUNK];
    __shared__ RowFacts facts[ROWS];
    __shared__ int paths[ROWS][WORDS], node_at[WORDS * 32];      // the rows' ancestors; where the tree's drafted tokens lie in the chunk, or -1
    pdl_launch_dependents();
    pdl_wait();
    const int lo = (int)blockIdx.x * CHUNK, n = min(CHUNK, A.vocab - lo), tid = threadIdx.x;
    const int r0 = (int)blockIdx.y * A.rows_per_block, rows = min(A.rows - r0, A.rows_per_block);
    if (tid < rows) {
        const int r = r0 + tid;
        RowFacts f;
        f.rep = A.penalties[3 * r];
        f.freq = A.penalties[3 * r + 1];
        f.pres = A.penalties[3 * r + 2];
        f.list = A.list_of_row ? A.list_of_row[r] : r;
        if (f.list < 0 || f.list >= A.lists) f.list = -1;
        f.mask = A.mask == nullptr ? -1 : (A.mask_of_row ? A.mask_of_row[r] : r);
        if (f.mask < 0 || f.mask >= A.masks) f.mask = -1;
        f.first = A.drafted ? A.first_row[r] : 0;
        f.bias = A.bias_start ? max(0, A.bias_start[r]) : 0;
        f.biases = A.bias_start ? (int)max(0LL, min((long long)A.bias_start[r + 1], A.bias_len) - f.bias) : 0;
        facts[tid] = f;
    }
    for (int i = tid; i < rows * A.words; i += THREADS) paths[i / A.words][i % A.words] = A.ancestors[(size_t)r0 * A.words + i];
    __syncthreads();
    float4 x[VECS];
    int may_word[VECS];
    // The row's logits that lie on 16-byte boundaries are taken four at a time, behind `head` (0 to 3) that do not; `whole` of them.
    int head = 0, whole = 0;
    auto fetch = [&](int k) {
        const float* in = A.logits + (size_t)(r0 + k) * A.in_stride + lo;
        head = min(n, (int)((16 - ((uintptr_t)in & 15)) & 15) / 4);
        whole = (n - head) / 4;
        const int* mask = facts[k].mask >= 0 ? A.mask + (size_t)facts[k].mask * A.mask_words : nullptr;
#pragma unroll
        for (int j = 0; j < VECS; ++j) {
            const int i = tid + j * THREADS;
            if (i < whole) {
                x[j] = __ldcs(reinterpret_cast<const float4*>(in + head) + i);
                if (mask) may_word[j] = mask[(lo + head + 4 * i) >> 5];
            }
        }
    };
    // adds `by` to the counts of the drafted tokens on the row's path
    auto add_path = [&](int k, unsigned by) {
        for (int i = tid; i < A.words * 32; i += THREADS)
            if ((paths[k][i >> 5] >> (i & 31) & 1) && node_at[i] >= 0) atomicAdd(&count[node_at[i]], by);
    };
    fetch(0);
    int counted = -2, tree = -1;               // the list that `count` holds (-1: none), the tree that `node_at` does
    for (int k = 0; k < rows; ++k) {
        const RowFacts f = facts[k];
        if (f.list != counted || (A.drafted && f.first != tree)) {
            __syncthreads();                   // (the last row's path has been taken away)
            if (f.list != counted) {
#pragma unroll
                for (int j = 0; j < VECS; ++j) reinterpret_cast<uint4*>(count)[tid + j * THREADS] = make_uint4(0u, 0u, 0u, 0u);
            }
            if (A.drafted && f.first != tree)
                for (int i = tid; i < A.words * 32; i += THREADS) {
                    const long long row = (long long)f.first + i;
                    const unsigned u = row >= 0 && row < A.rows ? (unsigned)(A.drafted[row] - lo) : 0xffffffffu;
                    node_at[i] = u < (unsigned)n ? (int)u : -1;
                }
            __syncthreads();
            if (f.list >= 0 && f.list != counted) {
                const long long a = max(0, A.history_start[f.list]), z = min((long long)A.history_start[f.list + 1], A.history_len);
                const long long said = a + A.prompt_len[f.list];
#pragma unroll 4
                for (long long i = a + tid; i < z; i += THREADS) {
                    const unsigned u = (unsigned)(A.history[i] - lo);
                    if (u < (unsigned)n) {
                        if (i < said) atomicOr(&count[u], ASKED);
                        else atomicAdd(&count[u], 1u);
                    }
                }
            }
            counted = f.list;
            tree = f.first;
        }
        if (A.drafted) add_path(k, 1u);
        const int bias_v = tid < f.biases ? A.bias_tokens[f.bias + tid] : -1;      // on its way while the row is worked on
        __syncthreads();
        const int* mask = f.mask >= 0 ? A.mask + (size_t)f.mask * A.mask_words : nullptr;
        const float* in = A.logits + (size_t)(r0 + k) * A.in_stride + lo;
        float* out = A.out + (size_t)(r0 + k) * A.out_stride + lo;
        const bool fours = (((uintptr_t)(out + head)) & 15) == 0;
        // (the few beside the fours)
        for (int i = tid; i < n - 4 * whole; i += THREADS) {
            const int u = i < head ? i : i + 4 * whole;
            const bool may = mask == nullptr || (mask[(lo + u) >> 5] >> ((lo + u) & 31) & 1);
            out[u] = may ? ruled(in[u], count[u], f.rep, f.freq, f.pres) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < VECS; ++j) {
            const int i = tid + j * THREADS, u = head + 4 * i;
            if (i >= whole) continue;
            uint4 c;
            if (head == 0) c = reinterpret_cast<const uint4*>(count)[i];
            else c = make_uint4(count[u], count[u + 1], count[u + 2], count[u + 3]);
            const int shift = (lo + u) & 31;
            unsigned may = mask ? (unsigned)may_word[j] >> shift : 15u;
            // four bits that begin in the last three of a word go on in the next one, which is there: a token's word is
            if (mask && shift > 28) may = __funnelshift_r((unsigned)may_word[j], (unsigned)mask[((lo + u) >> 5) + 1], shift);
            float4 y = x[j];
            if (c.x | c.y | c.z | c.w) {
                y.x = ruled(y.x, c.x, f.rep, f.freq, f.pres);
                y.y = ruled(y.y, c.y, f.rep, f.freq, f.pres);
                y.z = ruled(y.z, c.z, f.rep, f.freq, f.pres);
                y.w = ruled(y.w, c.w, f.rep, f.freq, f.pres);
            }
            if (!(may & 1u)) y.x = -INFINITY;
            if (!(may & 2u)) y.y = -INFINITY;
            if (!(may & 4u)) y.z = -INFINITY;
            if (!(may & 8u)) y.w = -INFINITY;
            if (fours) {
                reinterpret_cast<float4*>(out + head)[i] = y;
            } else {
                out[u] = y.x;
                out[u + 1] = y.y;
                out[u + 2] = y.z;
                out[u + 3] = y.w;
            }
        }
        if (k + 1 < rows) fetch(k + 1);
        if (!A.drafted && f.biases == 0) continue;
        __syncthreads();                       // the counts have been read, the row is written
        if (A.drafted) add_path(k, 0xffffffffu);
        // a token that several entries name gets their sum, in their order, from the thread of the first
        for (int i = tid; i < f.biases; i += THREADS) {
            const int* tokens = A.bias_tokens + f.bias;
            const int v = i == tid ? bias_v : tokens[i];
            const unsigned u = (unsigned)(v - lo);
            if (u >= (unsigned)n) continue;
            if (mask != nullptr && !(mask[v >> 5] >> (v & 31) & 1)) continue;
            bool first = true;
            for (int j = 0; j < i && first; ++j) first = tokens[j] != v;
            if (!first) continue;
            float y = out[u];
            for (int j = i; j < f.biases; ++j)
                if (tokens[j] == v) y += A.bias_values[f.bias + j];
            out[u] = y;
        }
    }
}

template <int VECS>
int launch(RuleArgs A, cudaStream_t stream) {
    const int chunks = (A.vocab + 4 * THREADS * VECS - 1) / (4 * THREADS * VECS);
    // rows that share a list are counted once where they follow each other in a block: as many rows to a block as leave eight blocks
    // for every processor
    const long long blocks = (long long)chunks * A.rows;
    A.rows_per_block = (int)(blocks / (148 * 8));
    A.rows_per_block = A.rows_per_block < 1 ? 1 : (A.rows_per_block > ROWS ? ROWS : A.rows_per_block);
    return xb_launch(logit_rules_kernel<VECS>, dim3(chunks, (A.rows + A.rows_per_block - 1) / A.rows_per_block), dim3(THREADS), 0, stream, A);
}

}  // namespace

XB_EXPORT int xb_logit_rules(float* out, const float* logits, const float* penalties, const int* history, const int* history_start, const int* prompt_len,
                             const int* list_of_row, const int* drafted, const int* ancestors, const int* first_row, const int* bias_start,
                             const int* bias_tokens, const float* bias_values, const int* mask, const int* mask_of_row, long long out_stride,
                             long long in_stride, long long history_len, long long bias_len, int rows, int lists, int vocab, int words, int masks,
                             int mask_words, cudaStream_t stream) {
    if (rows <= 0 || vocab <= 0) return 0;
    if (rows > (1 << 20) || words > WORDS || (mask && mask_words < (vocab + 31) / 32)) return (int)cudaErrorInvalidValue;
    const RuleArgs A{out, logits, penalties, history, history_start, prompt_len, list_of_row, drafted, ancestors, first_row, bias_start, bias_tokens,
                     bias_values, mask, mask_of_row, out_stride, in_stride, history_len, bias_len, rows, lists, vocab, words, masks, mask_words, 1};
    // chunks of 1,024 tokens while that leaves processors without work, of 4,096 when there are rows enough
    return (long long)rows * vocab < 148LL * 2 * 4096 ? launch<1>(A, stream) : launch<4>(A, stream);
}
