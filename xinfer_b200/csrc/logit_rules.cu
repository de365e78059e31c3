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
    int rows, lists, vocab, words, masks, mask_words;
};

// (`inv` is 1 / rep, rounded: a product in place of a quotient is one float32 rounding more, and a sixth of the instructions)
__device__ __forceinline__ float ruled(float x, unsigned count, float rep, float inv, float freq, float pres) {
    const unsigned c = count & ~ASKED;
    const float y = x * (x > 0.f ? inv : rep), z = c ? y - freq * (float)c - pres : y;      // (no branch: a warp nearly always has such a token)
    return count ? z : x;
}

constexpr int WARPS = THREADS / 32;
constexpr int ROWS = 48;                        // rows at a time: what they need to know lies in shared memory
constexpr int WORDS = 32;                       // words of ancestors: trees of up to 1,024 nodes
constexpr int NO_TREE = -32 * WORDS - 1;        // no row's tree: one that begins so far before the first row has no node, and all such are one
constexpr int BIASES = 192;                     // biases of these rows that lie in the chunk

struct __align__(16) RowFacts {
    float rep, inv, freq, pres;
    int list, mask, first, bias, biases;
    unsigned biased;                            // a bit per warp that has tokens with biases
};
struct Bias {
    int at, entry;                              // row << 16 | where in the chunk; which entry it is
    float value;                                // of all the row's entries for that token, in their order; in the first of them
    int first;                                  // whether it is that
};

template <int N>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}

constexpr int chunk_of(int vecs) { return 4 * THREADS * vecs; }
constexpr int mask_room(int vecs) { return WARPS * vecs * 5; }
constexpr int smem_of(int vecs, int words) { return 4 * (2 * chunk_of(vecs) + mask_room(vecs) + words * (ROWS + 4 * WARPS + 32)); }

// The vocabulary is cut into chunks of 1,024 VECS tokens, and the (chunk, row) pairs, chunk by chunk, into equal shares for as many blocks
// as the device holds.  The lists' tokens are counted in shared memory, once for rows that follow each other with one list (the nodes of a
// tree); a row's own path is added before it and taken away behind it.  A warp owns 128 of every 1,024 tokens, with their counts, mask
// words and biases, so that the warps of a block go through the rows without waiting for each other: while one waits for its next row, others
// work.  Which 128 these are goes by where a row starts, so rows of trees that do not all start alike on 16 bytes have a barrier between
// them: a count that one warp raises for its row may be another one's in the next.
// Bound by memory: a logit is read and written once.  512 rows of 151,936 with masks, biases and 8 histories of up to 4,096: 131 us, 4.75 TB/s (a
// copy of as many bytes takes 97); the rest is the blocks' start (a history is counted by every block that meets it) and four blocks a
// processor for want of registers.  In chunks of 2,048: 152 us.  Asking for a row before the one in front of it is worked on, into room of its
// own: 139 us; the blocks already have 64 KB a processor on their way, and more reads between the writes slow both.  512 rows of 151,935: 143
// us.  A single row of 151,936: 5.6 us, of which the launch and one trip for each of facts, history and logits are nearly all.
template <int VECS>
__global__ void __launch_bounds__(THREADS, 4)
logit_rules_kernel(const RuleArgs A) {
    constexpr int CHUNK = chunk_of(VECS);
    extern __shared__ __align__(16) unsigned count[];            // [CHUNK], then a row's logits and its mask words
    float4* const logits_at = reinterpret_cast<float4*>(count + CHUNK);
    int* const masks_at = reinterpret_cast<int*>(count + 2 * CHUNK);                       // [WARPS][VECS][5]
    __shared__ RowFacts facts[ROWS];
    __shared__ Bias biases[BIASES];
    __shared__ int found;
    // the rows' ancestors [ROWS][words]; the nodes whose tokens a warp owns, by `head` [WARPS][4][words]; where the tree's drafted tokens lie
    // in the chunk, or -1 [words][32]
    unsigned* const paths = reinterpret_cast<unsigned*>(masks_at + mask_room(VECS));
    unsigned* const own_nodes = paths + ROWS * A.words;
    int* const node_at = reinterpret_cast<int*>(own_nodes + WARPS * 4 * A.words);
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long units = (long long)((A.vocab + CHUNK - 1) / CHUNK) * A.rows;
    const long long from = units * blockIdx.x / gridDim.x, to = units * (blockIdx.x + 1) / gridDim.x;
    int lo = 0, n = 0, r0 = 0, rows = 0;       // the chunk's first token, its tokens; rows r0 .. r0 + rows - 1
    int listed = 0;                            // their biases in `biases` (-1: of a row by itself, more than fit)
    unsigned nodes_here = 0;                   // a bit per `head` at which the warp has drafted tokens of the tree
    int counted = -2, tree = NO_TREE;          // the list that `count` holds (-1: none), the tree that `node_at` does; of this chunk

    // The row's logits that lie on 16-byte boundaries are taken four at a time, behind `head` (0 to 3) that do not; `whole` fours.
    const bool on_fours = ((uintptr_t)A.logits & 15) == 0 && A.in_stride % 4 == 0;             // then there are none of these anywhere
    const bool owners_move = A.drafted && A.in_stride % 4 != 0;                                // `head` differs from row to row
    auto head_of = [&](int k) { return on_fours ? 0 : min(n, (int)((16 - ((uintptr_t)(A.logits + (size_t)(r0 + k) * A.in_stride + lo) & 15)) & 15) / 4); };
    // the warp that has element u of the chunk; the first one has those beside the fours
    auto owner = [&](int u, int head, int whole) { return u < head || u >= head + 4 * whole ? 0 : (u - head) >> 7 & (WARPS - 1); };
    const int mask_word = (((lane / 5) * 4 * THREADS + warp * 128) >> 5) + lane % 5;
    auto fetch = [&](int k) {
        const float* in = A.logits + (size_t)(r0 + k) * A.in_stride + lo;
        const int head = head_of(k), whole = (n - head) / 4;
        float4* to = logits_at + tid;
        const float4* from = reinterpret_cast<const float4*>(in + head) + tid;
#pragma unroll
        for (int j = 0; j < VECS; ++j)
            if (tid + j * THREADS < whole) copy_async<16>(to + j * THREADS, from + j * THREADS);
        if (facts[k].mask >= 0 && lane < 5 * VECS) {             // the words of the warp's 128 tokens in each 1,024: four, or five off a word's start
            const int word = (lo >> 5) + mask_word;              // (a head of up to three tokens stays in the word)
            if (word < A.mask_words) copy_async<4>(masks_at + warp * VECS * 5 + lane, A.mask + (size_t)facts[k].mask * A.mask_words + word);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // adds `by` to the counts of the drafted tokens on the row's path, the warp's own ones
    auto add_path = [&](int k, int head, unsigned by) {
        for (int w = 0; w < A.words; ++w)
            if ((paths[k * A.words + w] & own_nodes[(warp * 4 + head) * A.words + w]) >> lane & 1) atomicAdd(&count[node_at[w * 32 + lane]], by);
    };
    auto work = [&](int k) {
        const RowFacts f = facts[k];
        const int head = head_of(k), whole = (n - head) / 4;
        if (f.list != counted || (A.drafted && f.first != tree)) {           // (the same for the whole block)
            __syncthreads();
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
                auto say = [&](int token, long long i) {
                    const unsigned u = (unsigned)(token - lo);
                    if (u < (unsigned)n) {
                        if (i < said) atomicOr(&count[u], ASKED);
                        else atomicAdd(&count[u], 1u);
                    }
                };
                // four tokens at a time from the first 16-byte boundary on
                const long long a4 = min(z, a + (long long)((16 - ((uintptr_t)(A.history + a) & 15)) & 15) / 4), z4 = z - max(0LL, z - a4) % 4;
                if (a + tid < a4) say(A.history[a + tid], a + tid);
                if (z4 >= a4 && z4 + tid < z) say(A.history[z4 + tid], z4 + tid);
#pragma unroll 4
                for (long long i = a4 + 4 * tid; i < z4; i += 4 * THREADS) {
                    const int4 t = *reinterpret_cast<const int4*>(A.history + i);
                    say(t.x, i);
                    say(t.y, i + 1);
                    say(t.z, i + 2);
                    say(t.w, i + 3);
                }
            }
            if (A.drafted && f.first != tree) {
                nodes_here = 0;
                for (int h = 0; h < 4; ++h)                      // for every way that a row may lie
                    for (int w = 0; w < A.words; ++w) {
                        const int u = node_at[w * 32 + lane], head = min(n, h);
                        const unsigned mine = __ballot_sync(0xffffffffu, u >= 0 && owner(u, head, (n - head) / 4) == warp);
                        if (lane == 0) own_nodes[(warp * 4 + h) * A.words + w] = mine;
                        if (mine) nodes_here |= 1u << h;
                    }
            }
            __syncthreads();
            counted = f.list;
            tree = f.first;
        }
        const bool said_here = nodes_here >> head & 1u, biased_here = f.biased >> warp & 1u;
        if (said_here) add_path(k, head, 1u);
        asm volatile("cp.async.wait_group 0;" ::: "memory");     // this row is there
        __syncwarp();
        const float4* x = logits_at + tid;
        const int* mask = f.mask >= 0 ? masks_at + warp * VECS * 5 : nullptr;
        const int* far_mask = f.mask >= 0 ? A.mask + (size_t)f.mask * A.mask_words : nullptr;
        const float* in = A.logits + (size_t)(r0 + k) * A.in_stride + lo;
        float* out = A.out + (size_t)(r0 + k) * A.out_stride + lo;
        const bool fours = (((uintptr_t)(out + head)) & 15) == 0;
        auto all_four = [&](float4 y, const uint4& c, unsigned may) {
            if (c.x | c.y | c.z | c.w) {
                y.x = ruled(y.x, c.x, f.rep, f.inv, f.freq, f.pres);
                y.y = ruled(y.y, c.y, f.rep, f.inv, f.freq, f.pres);
                y.z = ruled(y.z, c.z, f.rep, f.inv, f.freq, f.pres);
                y.w = ruled(y.w, c.w, f.rep, f.inv, f.freq, f.pres);
            }
            if (!(may & 1u)) y.x = -INFINITY;
            if (!(may & 2u)) y.y = -INFINITY;
            if (!(may & 4u)) y.z = -INFINITY;
            if (!(may & 8u)) y.w = -INFINITY;
            return y;
        };
        auto may_say = [&](int u) { return far_mask == nullptr || (far_mask[(lo + u) >> 5] >> ((lo + u) & 31) & 1); };
        if (head == 0 && fours && n == CHUNK) {
            // a whole chunk on 16-byte boundaries: the same in a third of the instructions (lo is a multiple of 32)
            float4* out4 = reinterpret_cast<float4*>(out) + tid;
            const uint4* count4 = reinterpret_cast<const uint4*>(count) + tid;
            const int shift = 4 * lane & 31;
#pragma unroll
            for (int j = 0; j < VECS; ++j) __stcs(out4 + j * THREADS, all_four(x[j * THREADS], count4[j * THREADS], mask ? (unsigned)mask[j * 5 + (lane >> 3)] >> shift : 15u));
        } else {
            if (warp == 0)         // (the few beside the fours)
                for (int i = lane; i < n - 4 * whole; i += 32) {
                    const int u = i < head ? i : i + 4 * whole;
                    out[u] = may_say(u) ? ruled(in[u], count[u], f.rep, f.inv, f.freq, f.pres) : -INFINITY;
                }
#pragma unroll
            for (int j = 0; j < VECS; ++j) {
                const int i = tid + j * THREADS, u = head + 4 * i;
                if (i >= whole) continue;
                uint4 c;
                if (head == 0) c = reinterpret_cast<const uint4*>(count)[i];
                else c = make_uint4(count[u], count[u + 1], count[u + 2], count[u + 3]);
                unsigned may = 15u;
                if (mask) {            // (four bits that begin in the last three of a word go on in the next one)
                    const int word = ((lo + u) >> 5) - ((lo + head + j * 4 * THREADS + warp * 128) >> 5), shift = (lo + u) & 31;
                    may = (unsigned)mask[j * 5 + word] >> shift;
                    if (shift > 28) may = __funnelshift_r((unsigned)mask[j * 5 + word], (unsigned)mask[j * 5 + word + 1], shift);
                }
                const float4 y = all_four(x[j * THREADS], c, may);
                if (fours) {
                    reinterpret_cast<float4*>(out + head)[i] = y;
                } else {
                    out[u] = y.x;
                    out[u + 1] = y.y;
                    out[u + 2] = y.z;
                    out[u + 3] = y.w;
                }
            }
        }
        if (!said_here && !biased_here) return;
        __syncwarp();                          // the warp's counts have been read, its part of the row is written
        if (said_here) add_path(k, head, 0xffffffffu);
        if (biased_here && listed > 0)
            for (int i = lane; i < listed; i += 32) {
                const Bias b = biases[i];
                const int u = b.at & 0xffff;
                if (b.first && b.at >> 16 == k && owner(u, head, whole) == warp && may_say(u)) out[u] += b.value;
            }
        if (listed < 0)
            for (int i = lane; i < f.biases; i += 32) {
                const int* tokens = A.bias_tokens + f.bias;
                const int v = tokens[i], u = v - lo;
                if ((unsigned)u >= (unsigned)n || owner(u, head, whole) != warp || !may_say(u)) continue;
                bool mine = true;
                for (int j = 0; j < i && mine; ++j) mine = tokens[j] != v;
                if (!mine) continue;
                float sum = 0.f;
                for (int j = i; j < f.biases; ++j)
                    if (tokens[j] == v) sum += A.bias_values[f.bias + j];
                out[u] += sum;
            }
    };
    for (long long at = from; at < to; at += rows) {
        r0 = (int)(at % A.rows);
        rows = (int)min((long long)min(ROWS, A.rows - r0), to - at);
        if ((int)(at / A.rows) * CHUNK != lo || at == from) {
            lo = (int)(at / A.rows) * CHUNK;
            n = min(CHUNK, A.vocab - lo);
            counted = -2;
            tree = NO_TREE;
        }
        __syncthreads();                       // (the rows before are done with)
        if (tid < rows) {
            const int r = r0 + tid;
            RowFacts f;
            f.rep = A.penalties[3 * r];
            f.inv = 1.f / f.rep;
            f.freq = A.penalties[3 * r + 1];
            f.pres = A.penalties[3 * r + 2];
            f.list = A.list_of_row ? A.list_of_row[r] : r;
            if (f.list < 0 || f.list >= A.lists) f.list = -1;
            f.mask = A.mask == nullptr ? -1 : (A.mask_of_row ? A.mask_of_row[r] : r);
            if (f.mask < 0 || f.mask >= A.masks) f.mask = -1;
            f.first = A.drafted ? max(A.first_row[r], NO_TREE + 1) : 0;
            f.bias = A.bias_start ? (int)min((long long)max(0, A.bias_start[r]), A.bias_len) : 0;
            f.biases = A.bias_start ? (int)max(0LL, min((long long)A.bias_start[r + 1], A.bias_len) - f.bias) : 0;
            f.biased = 0u;
            facts[tid] = f;
        }
        for (int i = tid; i < rows * A.words; i += THREADS) paths[i] = A.ancestors[(size_t)r0 * A.words + i];
        if (tid == 0) found = 0;
        __syncthreads();
        fetch(0);
        listed = 0;
        while (A.bias_start) {
            // what the rows' entries say of tokens in the chunk; of fewer rows if that is more than there is room for
            const int first = facts[0].bias, entries = max(0, facts[rows - 1].bias + facts[rows - 1].biases - first);
            for (int i = tid; i < entries; i += THREADS) {
                const int u = A.bias_tokens[first + i] - lo;
                if ((unsigned)u >= (unsigned)n) continue;
                int row = 0, to_row = rows;        // (the last row that begins at or before the entry; rows without entries begin where the next does)
                while (to_row - row > 1) {
                    const int mid = (row + to_row) >> 1;
                    if (facts[mid].bias - first <= i) row = mid;
                    else to_row = mid;
                }
                const int at = facts[row].bias - first;
                if (i < at || i >= at + facts[row].biases) continue;        // (starts that do not ascend)
                const int slot = atomicAdd(&found, 1);
                if (slot < BIASES) biases[slot] = Bias{row << 16 | u, i, A.bias_values[first + i], 1};
            }
            __syncthreads();
            listed = found;
            if (listed <= BIASES) break;
            if (rows == 1) {
                listed = -1;
                break;
            }
            rows = (rows + 1) / 2;
            __syncthreads();
            if (tid == 0) found = 0;
            __syncthreads();
        }
        if (listed < 0) {
            if (tid == 0) facts[0].biased = 0xffffffffu;
            __syncthreads();
        }
        if (listed > 0) {
            // a token that several of a row's entries name gets their sum, in their order, by the first of them
            float sums[(BIASES + THREADS - 1) / THREADS];
#pragma unroll
            for (int x = 0; x < (BIASES + THREADS - 1) / THREADS; ++x) {
                const int i = tid + x * THREADS;
                if (i >= listed) continue;
                const Bias b = biases[i];
                int next = 0x7fffffff;             // the earliest entry behind b for the same token
                bool mine = true;
                for (int j = 0; j < listed; ++j) {
                    if (biases[j].at != b.at) continue;
                    if (biases[j].entry < b.entry) mine = false;
                    else if (biases[j].entry > b.entry) next = min(next, biases[j].entry);
                }
                sums[x] = b.value;
                while (mine && next != 0x7fffffff) {
                    int after = 0x7fffffff;
                    for (int j = 0; j < listed; ++j) {
                        if (biases[j].at != b.at) continue;
                        if (biases[j].entry == next) sums[x] += biases[j].value;
                        else if (biases[j].entry > next) after = min(after, biases[j].entry);
                    }
                    next = after;
                }
                biases[i].first = mine;
                if (mine) {
                    const int row = b.at >> 16, head = head_of(row);
                    atomicOr(&facts[row].biased, 1u << owner(b.at & 0xffff, head, (n - head) / 4));
                }
            }
            __syncthreads();                       // (the values have been read)
#pragma unroll
            for (int x = 0; x < (BIASES + THREADS - 1) / THREADS; ++x)
                if (tid + x * THREADS < listed) biases[tid + x * THREADS].value = sums[x];
            __syncthreads();
        }
        for (int k = 0; k < rows; ++k) {
            if (owners_move && k > 0) __syncthreads();     // the row before has taken its path's counts away, whosever they are now
            work(k);
            __syncwarp();                      // (the row lies where the warp's part of this one does)
            if (k + 1 < rows) fetch(k + 1);
        }
    }
}

template <int VECS>
int launch(const RuleArgs& A, cudaStream_t stream) {
    const int smem = smem_of(VECS, A.words);
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(logit_rules_kernel<VECS>, smem_of(VECS, WORDS), &roomy)) return rc;
    // as many blocks as the device holds: 228 KB of shared memory a processor, of which every block takes its own, the static arrays and 1 KB; four by their registers
    const int per_sm = (228 * 1024) / (smem + (int)(ROWS * sizeof(RowFacts) + BIASES * sizeof(Bias)) + 1024);
    const int resident = (per_sm < 1 ? 1 : (per_sm > 4 ? 4 : per_sm)) * 148;
    const long long units = (long long)((A.vocab + chunk_of(VECS) - 1) / chunk_of(VECS)) * A.rows;
    return xb_launch(logit_rules_kernel<VECS>, dim3((unsigned)(units < resident ? units : resident)), dim3(THREADS), smem, stream, A);
}

}  // namespace

static int logit_rules(float* out, const float* logits, const float* penalties, const int* history, const int* history_start, const int* prompt_len,
                       const int* list_of_row, const int* drafted, const int* ancestors, const int* first_row, const int* bias_start,
                       const int* bias_tokens, const float* bias_values, const int* mask, const int* mask_of_row, long long out_stride,
                       long long in_stride, long long history_len, long long bias_len, int rows, int lists, int vocab, int words, int masks,
                       int mask_words, cudaStream_t stream) {
    if (rows <= 0 || vocab <= 0) return 0;
    if (rows > (1 << 20) || words > WORDS || (mask && mask_words < (vocab + 31) / 32)) return (int)cudaErrorInvalidValue;
    const RuleArgs A{out, logits, penalties, history, history_start, prompt_len, list_of_row, drafted, ancestors, first_row, bias_start, bias_tokens,
                     bias_values, mask, mask_of_row, out_stride, in_stride, history_len, bias_len, rows, lists, vocab, words, masks, mask_words};
    // Chunks of 1,024 tokens while those of 4,096 would leave half of the processors without work.  Small and large chunks measured: one row of
    // 151,936 5.6 and 5.9 us, of 256,000 with 20,000 said 13.9 and 16.5; three rows of 151,936 6.8 and 6.3, four 8.2 and 6.6, seven 10.8 and 7.7.
    return (long long)rows * vocab < 148LL * 2048 ? launch<1>(A, stream) : launch<4>(A, stream);
}
XB_EXPORT int xb_logit_rules(const long long* words, int n) { return xb_by_words(logit_rules, words, n); }
