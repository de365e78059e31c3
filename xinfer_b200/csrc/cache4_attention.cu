// Attention of a step's tokens over a paged cache of 4-bit codes (codes4.cuh): token i of request b, at position lengths[b] - nodes + i, gets
//   sum_j softmax_j(scale q . k_j) v_j   over the keys j up to its position, of these the last `window`; zeros if it sees none.
// The step's own keys are in the cache already.  A page outside the pool is reported and its keys are not seen.
//
// Three kernels.  bfloat16, pages of a multiple of 8 tokens, heads of up to 128 channels or of 225 to 256: cache4_attention_mma.cu, which reads the keys once
// for 8 or 16 rows.  Requests of TC_ROWS rows (tokens times query heads of a key/value head) and more, heads of up to 128 channels, a scale above zero, pages whose
// bytes are a multiple of 16: cache4_attention_tc.cu, once for 256 rows (beside the first or the last, which takes what it leaves).  Everything else, float32 first of
// all: the one below.
#include "cache4_attention_mma.h"
#include "cache4_attention_tc.h"

namespace {

using namespace xb4;

// ---- any type and size -----------------------------------------------------------------------------------------------------
// A block per (16 rows, key/value head, request, share of the keys); the rows are (token, query head of the group) pairs.  A tile of 64 keys is
// taken out of its codes once for the 16 rows; products in float32, whose multiply-adds and their operands in shared memory bound it.  Shares so
// that two blocks have a processor; they are joined in their order by a second kernel.  Three requests of 13 tokens at up to 777 keys (window 256), 10 heads over 5 of 48
// channels, float32: 21 us; with every thread holding all 16 rows of two channels (as heads of more than 64 channels have them) 31 us.
constexpr int RT = 16, KT = 64, THREADS = 128, DIM_MOST = 256, SPLITS_MOST = 16, BLOCKS = 296;

__host__ __device__ constexpr int padded(int d) { return groups_of(d) * GROUP; }
constexpr int smem_bytes(int dp) { return 4 * (RT * dp + KT * (dp + 4) + KT * dp + RT * (KT + 1) + KT * RT + 3 * RT + 2 * KT); }

// Row r is token r / group of the request, query head r % group.  NARROW: heads of up to 64 channels.
template <typename T, int NARROW>
__global__ void __launch_bounds__(THREADS)
cache4_attention_any_kernel(const AttendArgs A, float* parts, int splits) {
    extern __shared__ __align__(16) float mem[];
    const int d = A.d, dp = padded(d), groups = groups_of(d), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* q = mem;                            // [RT][dp]
    float* k = q + RT * dp;                    // [KT][dp + 4]
    float* v = k + KT * (dp + 4);              // [KT][dp]
    float* s = v + KT * dp;                    // [RT][KT + 1]
    float* p = s + RT * (KT + 1);              // [KT][RT]; below zero: not seen
    float* m = p + KT * RT;                    // [RT]: maximum so far, sum so far, what the sums so far are multiplied by
    float* l = m + RT;
    float* alpha = l + RT;
    int* page = reinterpret_cast<int*>(alpha + RT);      // [KT]: a key's page, -1 without one
    int* place = page + KT;
    pdl_overlap_few();
    const int b = blockIdx.y, g = blockIdx.x % A.nkv, group = A.group, step = gridDim.x / A.nkv;
    const Request r = request_of<true>(A, b);
    const int rows = r.nodes * group;
    for (int rt = blockIdx.x / A.nkv; rt * RT < rows; rt += step) {
        const int row0 = rt * RT, many = min(RT, rows - row0);
        const int pos0 = r.first_pos + row0 / group, pos1 = r.first_pos + (row0 + many - 1) / group;
        const int lo = first_seen(A, pos0) / KT, hi = (min(pos1 + 1, r.keys) + KT - 1) / KT, tiles = max(0, hi - lo);
        const int from = lo + (int)((long long)tiles * blockIdx.z / splits), to = lo + (int)((long long)tiles * (blockIdx.z + 1) / splits);
        auto row_of = [&](int i, long long stride) { return (r.first + (row0 + i) / group) * stride + (long long)(g * group + (row0 + i) % group) * d; };
        for (int i = tid; i < RT * dp; i += THREADS) {
            const int y = i / dp, c = i % dp;
            q[i] = y < many && c < d ? to_f32<T>(static_cast<const T*>(A.q)[row_of(y, A.q_stride) + c]) : 0.f;
        }
        if (tid < RT) m[tid] = -INFINITY, l[tid] = 0.f;
        // sums: a thread has a channel and all rows, or (heads of up to 64 channels) half of the rows
        constexpr int CHANNELS = NARROW ? 1 : DIM_MOST / THREADS, MINE = NARROW ? RT / 2 : RT;
        const int own = NARROW ? tid % 64 : tid, rows0 = NARROW ? tid / 64 * MINE : 0;
        float acc[CHANNELS][MINE] = {};
        __syncthreads();
        for (int tile = from; tile < to; ++tile) {
            if (tid < KT) {
                const int key = tile * KT + tid;
                int id = -1;
                if (key < r.keys && key <= pos1 && key >= first_seen(A, pos0)) {
                    id = A.block_table[(long long)b * A.table_stride + key / A.page_size];
                    if (id < 0 || id >= A.num_pages) {
                        atomicOr(A.err, XB_ERR_BAD_PAGE);
                        id = -1;
                    }
                }
                page[tid] = id;
                place[tid] = key % A.page_size;
            }
            __syncthreads();
            bool strange = false;              // a value's group is no number: what does not see it must not add zero times that
            for (int i = tid; i < 2 * KT * groups; i += THREADS) {
                const int key = i % KT, j = i / KT % groups;
                const bool is_k = i < KT * groups;
                uint32_t code[4] = {0, 0, 0, 0}, word = 0;
                if (page[key] >= 0) {
                    const uint8_t* from_page = (is_k ? A.k_cache : A.v_cache) + ((long long)page[key] * A.nkv + g) * ((long long)A.page_size * row_bytes(d));
                    const uint32_t* c4 = reinterpret_cast<const uint32_t*>(from_page + ((long long)j * A.page_size + place[key]) * GROUP_BYTES);
#pragma unroll
                    for (int e = 0; e < 4; ++e) code[e] = c4[e];
                    word = reinterpret_cast<const uint32_t*>(from_page + (long long)groups * A.page_size * GROUP_BYTES)[place[key] * groups + j];
                }
                strange |= !is_k && !(fabsf(scale_of(word)) < INFINITY && fabsf(least_of(word)) < INFINITY);
                float* to_row = is_k ? k + key * (dp + 4) + j * GROUP : v + key * dp + j * GROUP;
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const uint32_t c = code[e / 8] >> (4 * (e & 7));
                    // (channels behind the head have codes nobody wrote: the queries there are zero, and so are the keys)
                    const int left = d - (j * GROUP + e);
                    float4 x;
                    x.x = left > 0 ? value_of(c & 15, word) : 0.f;
                    x.y = left > 1 ? value_of(c >> 4 & 15, word) : 0.f;
                    x.z = left > 2 ? value_of(c >> 8 & 15, word) : 0.f;
                    x.w = left > 3 ? value_of(c >> 12 & 15, word) : 0.f;
                    *reinterpret_cast<float4*>(to_row + e) = x;
                }
            }
            strange = __syncthreads_or(strange);
            {
                const int key = tid % KT, y0 = tid / KT * (RT / 2);
                float sum[RT / 2] = {};
                for (int c = 0; c < dp; c += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(k + key * (dp + 4) + c);
#pragma unroll
                    for (int y = 0; y < RT / 2; ++y) {
                        const float4 z = *reinterpret_cast<const float4*>(q + (y0 + y) * dp + c);
                        sum[y] = fmaf(x.x, z.x, fmaf(x.y, z.y, fmaf(x.z, z.z, fmaf(x.w, z.w, sum[y]))));
                    }
                }
#pragma unroll
                for (int y = 0; y < RT / 2; ++y) s[(y0 + y) * (KT + 1) + key] = sum[y] * A.scale;
            }
            __syncthreads();
            for (int y = warp; y < RT; y += THREADS / 32) {
                const int pos = r.first_pos + (row0 + y) / group, low = first_seen(A, pos);
                bool seen[2];
                float x[2], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int at = lane + 32 * e, key = tile * KT + at;
                    seen[e] = y < many && page[at] >= 0 && key <= pos && key >= low;
                    x[e] = s[y * (KT + 1) + at];
                    if (seen[e]) top = max_nan(top, x[e]);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float old = m[y], now = max_nan(old, top), base = now == -INFINITY ? 0.f : now;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float w = expf(x[e] - base);
                    p[(lane + 32 * e) * RT + y] = seen[e] ? w : (strange ? -1.f : 0.f);
                    if (seen[e]) sum += w;
                }
                sum = warp_sum(sum);
                __syncwarp();
                if (lane == 0) {
                    const float a = old == -INFINITY ? 0.f : expf(old - base);
                    alpha[y] = a;
                    m[y] = now;
                    l[y] = l[y] * a + sum;
                }
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < CHANNELS; ++e) {
                const int c = own + e * THREADS;
                if (c >= dp) break;
#pragma unroll
                for (int y = 0; y < MINE; ++y) acc[e][y] *= alpha[rows0 + y];         // (what is no number stays so, however far below a later score it is)
#pragma unroll 2
                for (int key = 0; key < KT; ++key) {
                    const float x = v[key * dp + c];
                    float w[MINE];
#pragma unroll
                    for (int y = 0; y < MINE; y += 4) *reinterpret_cast<float4*>(w + y) = *reinterpret_cast<const float4*>(p + key * RT + rows0 + y);
                    if (!strange) {
#pragma unroll
                        for (int y = 0; y < MINE; ++y) acc[e][y] = fmaf(w[y], x, acc[e][y]);
                    } else {
#pragma unroll
                        for (int y = 0; y < MINE; ++y)
                            if (!(w[y] < 0.f)) acc[e][y] = fmaf(w[y], x, acc[e][y]);
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < CHANNELS; ++e) {
            const int c = own + e * THREADS;
            if (c >= d) break;
#pragma unroll
            for (int j = 0; j < MINE; ++j) {
                const int y = rows0 + j;
                if (y >= many) break;
                if (splits == 1) {
                    static_cast<T*>(A.out)[row_of(y, A.out_stride) + c] = from_f32<T>(l[y] == 0.f ? 0.f : acc[e][j] / l[y]);
                } else {
                    float* to_part = parts + ((long long)blockIdx.z * A.tokens * A.nh + row_of(y, (long long)A.nh * d) / d) * (d + 2);
                    to_part[c] = acc[e][j];
                    if (c == 0) to_part[d] = m[y], to_part[d + 1] = l[y];
                }
            }
        }
        __syncthreads();
    }
}

// A warp per row: its parts, each with the maximum and the sum that it was formed with.
template <typename T>
__global__ void __launch_bounds__(THREADS)
cache4_attention_any_join_kernel(const AttendArgs A, const float* parts, int splits) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)A.tokens * A.nh, row = (long long)blockIdx.x * (THREADS / 32) + threadIdx.x / 32;
    const int t = (int)(row / A.nh);
    // (rows behind the last request have no parts and stay as they are)
    if (row >= rows || t < A.token_start[0] || t >= A.token_start[A.requests]) return;
    float top = -INFINITY, total = 0.f;
    for (int i = 0; i < splits; ++i) top = max_nan(top, parts[(i * rows + row) * (A.d + 2) + A.d]);
    const float base = top == -INFINITY ? 0.f : top;
    float acc[DIM_MOST / 32] = {};
    for (int i = 0; i < splits; ++i) {
        const float* part = parts + (i * rows + row) * (A.d + 2);
        if (part[A.d] == -INFINITY) continue;
        const float f = expf(part[A.d] - base);
        total += f * part[A.d + 1];
#pragma unroll
        for (int e = 0; e < DIM_MOST / 32; ++e)
            if (lane + 32 * e < A.d) acc[e] = fmaf(f, part[lane + 32 * e], acc[e]);
    }
    T* out = static_cast<T*>(A.out) + t * A.out_stride + (row % A.nh) * A.d;
#pragma unroll
    for (int e = 0; e < DIM_MOST / 32; ++e)
        if (lane + 32 * e < A.d) out[lane + 32 * e] = from_f32<T>(total == 0.f ? 0.f : acc[e] / total);
}

struct AnyGrid {
    int row_tiles, splits;
};
AnyGrid any_grid(int requests, int nh, int nkv, int longest) {
    const long long tiles = ((longest < 1 ? 1 : longest) * (long long)(nh / nkv) + RT - 1) / RT;       // (a block takes more than one where they are more)
    AnyGrid g;
    g.row_tiles = tiles > 4096 ? 4096 : (int)tiles;
    const long long s = BLOCKS / ((long long)g.row_tiles * nkv * requests);
    g.splits = s < 1 ? 1 : (s > SPLITS_MOST ? SPLITS_MOST : (int)s);
    return g;
}

template <typename T>
int launch_any(const AttendArgs& A, int longest, float* scratch, cudaStream_t stream) {
    AnyGrid g = any_grid(A.requests, A.nh, A.nkv, longest);
    if (A.wide) g.splits = 1;                  // (for requests that another kernel has left: there is no scratch for shares)
    static unsigned long long roomy[2] = {0, 0};
    const bool narrow = padded(A.d) <= 64;
    auto go = [&](auto kernel, unsigned long long* done) {
        if (const int rc = xb_more_smem(kernel, smem_bytes(DIM_MOST), done)) return rc;
        return xb_launch_few(kernel, dim3(g.row_tiles * A.nkv, A.requests, g.splits), dim3(THREADS), smem_bytes(padded(A.d)), stream, A, scratch, g.splits);
    };
    const int rc = narrow ? go(cache4_attention_any_kernel<T, 1>, &roomy[0]) : go(cache4_attention_any_kernel<T, 0>, &roomy[1]);
    if (rc || g.splits == 1) return rc;
    const long long rows = (long long)A.tokens * A.nh;
    return xb_launch(cache4_attention_any_join_kernel<T>, dim3((unsigned)((rows + THREADS / 32 - 1) / (THREADS / 32))), dim3(THREADS), 0, stream, A, scratch, g.splits);
}

}  // namespace

static int cache4_attention(int dtype, void* out, const void* q, const uint8_t* k_cache, const uint8_t* v_cache, const int* lengths, const int* token_start,
                            const int* block_table, long long out_stride, long long q_stride, int tokens, int requests, int table_stride, int nh, int nkv,
                            int d, int page_size, int num_pages, int window, int longest, float scale, float* scratch, int* err, cudaStream_t stream) {
    if (tokens <= 0 || requests <= 0) return 0;
    if (requests > REQUESTS_MAX || d < 1 || d > DIM_MOST || nkv < 1 || nh < nkv || nh % nkv || page_size < 1 || (long long)page_size * row_bytes(d) > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    if ((long long)table_stride * page_size > KEYS_MOST || (long long)tokens * nh > ROWS_MOST) return (int)cudaErrorInvalidValue;
    AttendArgs A{out, q, k_cache, v_cache, lengths, token_start, block_table, out_stride, q_stride, tokens, requests, table_stride, nh, nkv, d, page_size,
                       num_pages, window, nh / nkv, ((1ull << 32) + (unsigned)(nh / nkv) - 1) / (unsigned)(nh / nkv), 0, 0x7fffffff, scale, err, nullptr};
    if (dtype == XB_BF16 && tc_takes(A, longest)) {
        // requests of few rows beside those of many have the kernel for few (each reads on the device which requests are its own), which also takes what the
        // one for many leaves; where it does not take such pages the general one does
        const bool both = mma_takes(A);
        A.rows_from = both ? OWN_ROWS : 0;
        if (const int rc = tc_launch(A, scratch, stream)) return rc;
        A.rows_from = 0, A.rows_to = both ? OWN_ROWS : 0, A.wide = tc_wide(d, scratch);
        return both ? mma_launch(A, OWN_ROWS, scratch + tc_scratch(d), stream) : launch_any<__nv_bfloat16>(A, longest, nullptr, stream);
    }
    if (dtype == XB_BF16 && mma_takes(A)) return mma_launch(A, (nh / nkv) * (long long)longest > TC_ROWS ? TC_ROWS : (nh / nkv) * longest, scratch, stream);
    return dtype == XB_F32 ? launch_any<float>(A, longest, scratch, stream) : launch_any<__nv_bfloat16>(A, longest, scratch, stream);
}
XB_EXPORT int xb_cache4_attention(const long long* words, int n) { return xb_by_words(cache4_attention, words, n); }

// float32 numbers of scratch for a step
XB_EXPORT long long xb_cache4_attention_scratch(int dtype, int tokens, int requests, int nh, int nkv, int d, int longest) {
    if (tokens <= 0 || requests <= 0 || nkv <= 0 || nh < nkv || d < 1) return 0;
    const AnyGrid g = any_grid(requests, nh, nkv, longest);
    // (pages and scale are not known here: enough for any of the kernels)
    const long long any = g.splits == 1 ? 0 : (long long)g.splits * tokens * nh * (d + 2);
    const bool tc = dtype == XB_BF16 && tc_takes(nh, nkv, d, longest);
    const long long rows = (long long)(nh / nkv) * longest, few = dtype == XB_BF16 && mma_takes(d) ? mma_scratch(d, rows > TC_ROWS ? TC_ROWS : (int)rows) : 0, both = few + (tc ? tc_scratch(d) : 0);
    return any > both ? any : both;
}
