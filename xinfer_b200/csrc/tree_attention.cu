// Attention of a tree of drafted tokens over the paged cache.  Request b has `context[b]` cached keys and the nodes
// token_start[b] .. token_start[b + 1] - 1, whose keys and values lie in rows of their own beside the cache.  With scale s, node
// i of depth p_i sees the keys
//     cached j < context[b]                          (window w: and j > context[b] + p_i - w)
//     drafted i' with bit i' of ancestors[i] set     (window w: and p_i - p_i' < w)
// and its result is  sum_j exp(s q.k_j - m) v_j / sum_j exp(s q.k_j - m),  m the largest score;  zeros where it sees no key.
// A value that a node does not see is not part of its result, whatever it holds.
#include "tree_attention.cuh"

namespace {

using namespace xbtree;

// The kernel for float32, and for what the tcgen05 kernel does not take (tree_attention_tc.cu): any head size, group and page.  A job's rows
// are 32 (node, query head) pairs; a tile is 32 keys.  Scores are formed 2 rows x 4 keys a thread and values summed 4 rows x 4 channels at a
// time, by float32 multiply-adds from shared memory; four lanes form the softmax of a row, eight keys each.  Jobs, tiles and the join are
// those of the line in tree_attention.cuh, four blocks to a processor.  Bound by the multiply-adds and their operands from shared memory (six
// reads of four numbers for 32 multiply-adds): 8 trees of 64 nodes at up to 1,024 keys (32 heads over 8 of 128) 178 us, of which 5.6 GFLOP at
// the multiply-adds' rate are 75; 32 of 16 at up to 2,000 305 us.  Few tokens are bound by trips: three trees of 13 at 777 keys with a window (10
// heads over 5 of 48) 17 us: 2.2 until the first job is known, 1.2 pages and queries, 1.3 the tile, 2.1 its products, 0.7 the part, then the join.
constexpr int RT = 32, KT = 32, THREADS = 128, LINE_BLOCKS = 4 * 148;

// Four channels of a row from c on, zeros from d on; `fours`: rows start where four numbers may be read at once (and d is a multiple of 4).
__device__ __forceinline__ float4 four_of(const float* row, int c, int d, bool fours) {
    if (fours) return c < d ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(c < d ? row[c] : 0.f, c + 1 < d ? row[c + 1] : 0.f, c + 2 < d ? row[c + 2] : 0.f, c + 3 < d ? row[c + 3] : 0.f);
}
__device__ __forceinline__ float4 four_of(const __nv_bfloat16* row, int c, int d, bool fours) {
    if (fours) {
        if (c >= d) return make_float4(0.f, 0.f, 0.f, 0.f);
        const uint2 v = *reinterpret_cast<const uint2*>(row + c);
        return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
    }
    auto at = [&](int i) { return c + i < d ? __bfloat162float(row[c + i]) : 0.f; };
    return make_float4(at(0), at(1), at(2), at(3));
}
// The larger of two; one that is no number wins.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ bool finite(const float4& v) {
    return fabsf(v.x) <= 3.402823466e38f && fabsf(v.y) <= 3.402823466e38f && fabsf(v.z) <= 3.402823466e38f && fabsf(v.w) <= 3.402823466e38f;
}

// DP: the head size rounded up; rows of zeros lie behind d.
template <typename T, int DP>
__global__ void __launch_bounds__(THREADS)
tree_attention_kernel(const TreeArgs A, const Line line) {
    constexpr int LD = DP + 4, LP = KT + 4, CJ = DP / 64;
    extern __shared__ __align__(16) float smem[];
    float* const q_sm = smem;                      // [RT][LD]
    float* const k_sm = q_sm + RT * LD;            // [KT][LD]
    float* const v_sm = k_sm + KT * LD;            // [KT][DP]
    float* const p_sm = v_sm + KT * DP;            // [RT][LP]
    __shared__ Walk walk;
    __shared__ float corr[RT], sums[RT], tops[RT];
    __shared__ unsigned seen_of[RT];
    __shared__ long long rows_of[2][KT];           // of this tile and the next: where the keys begin in their tensor (-1: nowhere)
    __shared__ int depths[2][KT];                  // and their depths
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = A.nh / A.nkv;
    const T *q = (const T*)A.q, *k_new = (const T*)A.k_new, *v_new = (const T*)A.v_new, *k_cache = (const T*)A.k_cache, *v_cache = (const T*)A.v_cache;
    auto on_fours = [](const void* p, long long stride) { return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0 && stride % 4 == 0; };
    const bool fours = A.d % 4 == 0 && on_fours(q, A.q_stride) && on_fours(k_new, A.k_stride) && on_fours(v_new, A.v_stride) && on_fours(k_cache, 0) && on_fours(v_cache, 0);
    if (warp == 0) {
        const Walk w = place_in_line<KT>(A, line);
        if (lane == 0) walk = w;
    }
    __syncthreads();
    Walk w = walk;
    int told_of = 0;
    for (bool first = true; next_segment<KT>(A, line, w, first); first = false) {
        const RequestLine& s = w.r;
        const int row0 = w.piece * RT, rows = min(RT, s.nodes * G - row0);
        const bool whole = w.i1 - w.i0 == s.tiles;
        if (tid < RT) {
            tops[tid] = -INFINITY;
            sums[tid] = 0.f;
        }
        const int* table = A.block_table + (size_t)w.b * A.table_stride;
        float o[4][CJ][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < CJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][j][e] = 0.f;
        const int o_row = tid / 16 * 4, o_col = tid % 16 * 4;
        // a window's first key, of the root; keys before it are nobody's
        const int lo = A.window > 0 ? max(0, s.context - A.window + 1) : 0;
        // What a tile needs to know, of its keys by the first warp, a key to a lane, and of a row by the row's lanes: asked for while another
        // tile is worked on, then written down.
        const int my_row = tid >> 2, my_t = s.first + (row0 + min(my_row, rows - 1)) / G;
        const int my_depth = A.window > 0 ? max(0, A.depth[my_t]) : 0;
        int asked_page = 0, asked_depth = 0;
        unsigned asked_mask = 0;
        auto first_key = [&](int it) { return (it >= s.old_tiles ? it - s.old_tiles : s.tile0 + it) * KT; };
        auto ask = [&](int it) {
            const int key = first_key(it) + lane;
            const bool drafted = it >= s.old_tiles;
            asked_mask = 0;
            if (drafted && key / KT < A.words) asked_mask = (unsigned)A.ancestors[(size_t)my_t * A.words + key / KT];
            if (warp > 0) return;
            asked_page = asked_depth = 0;
            if (drafted) {
                if (A.window > 0 && key < s.nodes) asked_depth = max(0, A.depth[s.first + key]);
            } else if (key < s.context && key >= lo) {
                asked_page = table[key / A.page_size];
            }
        };
        auto write_down = [&](int it) {            // (the first warp)
            const int key = first_key(it) + lane;
            long long at = -1;
            if (it >= s.old_tiles) {
                if (key < s.nodes) at = s.first + key;
            } else if (key < s.context && key >= lo) {
                if (asked_page >= 0 && asked_page < A.num_pages) at = (((long long)asked_page * A.nkv + w.g) * A.page_size + key % A.page_size) * A.d;
                else atomicOr(A.err, XB_ERR_BAD_PAGE);
            }
            rows_of[it & 1][lane] = at;
            depths[it & 1][lane] = asked_depth;
        };
        ask(w.i0);
#pragma unroll 4
        for (int i = tid; i < RT * DP / 4; i += THREADS) {
            const int r = i / (DP / 4), c = i % (DP / 4) * 4, row = row0 + r;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) x = four_of(q + (size_t)(s.first + row / G) * A.q_stride + (size_t)(w.g * G + row % G) * A.d, c, A.d, fours);
            *reinterpret_cast<float4*>(q_sm + r * LD + c) = x;
        }
        unsigned my_mask = asked_mask;
        if (warp == 0) write_down(w.i0);
        for (int it = w.i0; it < w.i1; ++it) {
            const bool drafted = it >= s.old_tiles;
            const int key0 = drafted ? (it - s.old_tiles) * KT : (s.tile0 + it) * KT, keys = min(KT, (drafted ? s.nodes : s.context) - key0);
            bool odd = false;
            __syncthreads();                       // the tile before has been read
#pragma unroll 8
            for (int i = tid; i < KT * DP / 4; i += THREADS) {
                const int j = i / (DP / 4), c = i % (DP / 4) * 4;
                const long long at = rows_of[it & 1][j];
                float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
                if (at >= 0) {
                    k = four_of(drafted ? k_new + at * A.k_stride + (size_t)w.g * A.d : k_cache + at, c, A.d, fours);
                    v = four_of(drafted ? v_new + at * A.v_stride + (size_t)w.g * A.d : v_cache + at, c, A.d, fours);
                }
                odd |= !finite(v);
                *reinterpret_cast<float4*>(k_sm + j * LD + c) = k;
                *reinterpret_cast<float4*>(v_sm + j * DP + c) = v;
            }
            // a value that is not finite may be one that not all rows see: their weights of zero must not meet it
            const bool some_odd = __syncthreads_or(odd) && (drafted || A.window > 0);
            if (it + 1 < w.i1) ask(it + 1);
            {
                const int r = tid / 8 * 2, j = tid % 8;
                float sc[2][4] = {};
#pragma unroll 4
                for (int c = 0; c < DP; c += 4) {
                    float4 a[2], b[4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) a[x] = *reinterpret_cast<const float4*>(q_sm + (r + x) * LD + c);
#pragma unroll
                    for (int y = 0; y < 4; ++y) b[y] = *reinterpret_cast<const float4*>(k_sm + (j + 8 * y) * LD + c);
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            sc[x][y] = fmaf(a[x].x, b[y].x, sc[x][y]);
                            sc[x][y] = fmaf(a[x].y, b[y].y, sc[x][y]);
                            sc[x][y] = fmaf(a[x].z, b[y].z, sc[x][y]);
                            sc[x][y] = fmaf(a[x].w, b[y].w, sc[x][y]);
                        }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int y = 0; y < 4; ++y) p_sm[(r + x) * LP + j + 8 * y] = sc[x][y];
            }
            __syncthreads();
            {
                // which keys of the tile the row sees
                unsigned m = keys < 32 ? (1u << keys) - 1u : 0xffffffffu;
                if (my_row >= rows) m = 0;
                const int q8 = (tid & 3) * 8;
                if (drafted) {
                    m &= my_mask;
                    if (A.window > 0)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (my_depth - depths[it & 1][q8 + i] >= A.window) m &= ~(1u << (q8 + i));
                } else if (A.window > 0) {
                    const int from = s.context + my_depth - A.window + 1 - key0;
                    if (from > 0) m = from < 32 ? m & (0xffffffffu << from) : 0u;
                }
                float* p = p_sm + my_row * LP + q8;
                float x[8], top = -INFINITY;
                *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
                *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = m >> (q8 + i) & 1u ? x[i] * A.scale : -INFINITY;
                    top = max_nan(top, x[i]);
                }
                const float before = tops[my_row];
                top = max_nan(top, before);        // (a score that is no number makes the row one)
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float base = top == -INFINITY ? 0.f : top;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = expf(x[i] - base);
                    sum += x[i];
                }
                *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
                *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(x + 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                // (with a window the row's lanes have each looked at their own keys)
                unsigned seen = m & 0xffu << q8;
                seen |= __shfl_xor_sync(0xffffffffu, seen, 1);
                seen |= __shfl_xor_sync(0xffffffffu, seen, 2);
                if ((tid & 3) == 0) {
                    const float f = expf(before - base);
                    corr[my_row] = f;
                    sums[my_row] = sums[my_row] * f + sum;
                    tops[my_row] = top;
                    seen_of[my_row] = seen;
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float f = corr[o_row + r];
#pragma unroll
                for (int j = 0; j < CJ; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[r][j][e] *= f;
            }
            my_mask = asked_mask;
            if (warp == 0 && it + 1 < w.i1) write_down(it + 1);
            if (!some_odd) {
#pragma unroll 2
                for (int key = 0; key < KT; key += 4) {
                    float4 p[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[r] = *reinterpret_cast<const float4*>(p_sm + (o_row + r) * LP + key);
#pragma unroll
                    for (int y = 0; y < 4; ++y)
#pragma unroll
                        for (int j = 0; j < CJ; ++j) {
                            const float4 v = *reinterpret_cast<const float4*>(v_sm + (key + y) * DP + o_col + 64 * j);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float w = y == 0 ? p[r].x : y == 1 ? p[r].y : y == 2 ? p[r].z : p[r].w;
                                o[r][j][0] = fmaf(w, v.x, o[r][j][0]);
                                o[r][j][1] = fmaf(w, v.y, o[r][j][1]);
                                o[r][j][2] = fmaf(w, v.z, o[r][j][2]);
                                o[r][j][3] = fmaf(w, v.w, o[r][j][3]);
                            }
                        }
                }
            } else {
                for (int key = 0; key < KT; ++key)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (!(seen_of[o_row + r] >> key & 1u)) continue;
                        const float w = p_sm[(o_row + r) * LP + key];
#pragma unroll
                        for (int j = 0; j < CJ; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[r][j][e] = fmaf(w, v_sm[key * DP + o_col + 64 * j + e], o[r][j][e]);
                    }
            }
        }
        __syncthreads();
        const int which = w.i0 > 0 ? 0 : 1;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + o_row + r;
            if (o_row + r >= rows) continue;
            const float sum = sums[o_row + r], inv = whole ? (sum > 0.f || sum != sum ? 1.f / sum : 0.f) : 1.f;
            const size_t part = part_row(line, blockIdx.x, which, o_row + r);
            T* out = (T*)A.out + (size_t)(s.first + row / G) * A.out_stride + (size_t)(w.g * G + row % G) * A.d;
#pragma unroll
            for (int j = 0; j < CJ; ++j) {
                const int c0 = o_col + 64 * j;
                if (!whole && A.d % 4 == 0) {
                    if (c0 < A.d) *reinterpret_cast<float4*>(line.part_o + part * A.d + c0) = make_float4(o[r][j][0], o[r][j][1], o[r][j][2], o[r][j][3]);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c0 + e >= A.d) continue;
                    if (whole) out[c0 + e] = from_f32<T>(o[r][j][e] * inv);
                    else line.part_o[part * A.d + c0 + e] = o[r][j][e];
                }
            }
        }
        if (!whole) {
            if (tid < rows) {
                float* ml = line.part_ml + part_row(line, blockIdx.x, which, tid) * 2;
                ml[0] = tops[tid];
                ml[1] = sums[tid];
            }
            if (tid == 0) {
                int from;
                const int parts = job_parts(w, from);
                int* job = line.shared_jobs + (blockIdx.x * 2 + which) * 8;
                job[0] = parts;
                job[1] = from;
                job[2] = row0;
                job[3] = rows;
                job[4] = w.g;
                job[5] = s.first;
            }
            told_of |= 1 << which;
        }
        __syncthreads();                           // what the next job writes has been read
    }
    if (tid < 2 && !(told_of >> tid & 1)) line.shared_jobs[(blockIdx.x * 2 + tid) * 8] = 0;
}

// Joins the parts of a job that several blocks shared, in an order that does not change: with M the largest of their maxima,
// out = sum_i e^(m_i - M) O_i / sum_i e^(m_i - M) l_i.  A block per part, which takes as many of the job's rows.  Bound by trips to the L2: a warp
// has eight pieces of rows on their way, of several rows where a job has few parts, and asks for them before it forms their factors; of a job
// of more than eight parts the block's warps take a row together, every fourth part each.  3 us for 15 jobs in 7 parts, 4.5 us for 8 jobs in 65
// parts (a warp a row, four parts on their way: 4 and 11 us).
constexpr int JOIN_WARPS = THREADS / 32, JOIN_TOGETHER = 8;

struct JoinJob {
    int parts, c_first, row0, rows, g, first, G;
};

// `V` numbers of a row from c on (a row's numbers lie on its own, d a multiple of V or not).
template <int V>
__device__ __forceinline__ void piece_of(float* to, const float* row, int c, int d) {
    if (d % V == 0) {
        if constexpr (V == 4) {
            const float4 x = c < d ? __ldcg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
            to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
        } else {
            const float2 x = c < d ? __ldcg(reinterpret_cast<const float2*>(row + c)) : make_float2(0.f, 0.f);
            to[0] = x.x, to[1] = x.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) to[e] = c + e < d ? __ldcg(row + c + e) : 0.f;
    }
}

// P parts of R rows at a time by a warp; TOGETHER: one row by all warps.
template <typename T, int DP, int P, bool TOGETHER>
__device__ __forceinline__ void join_rows(const TreeArgs& A, const Line& line, const JoinJob& job, int r0, int r1) {
    constexpr int V = DP >= 128 ? 4 : 2, K = DP / (32 * V), R = TOGETHER || 8 / (P * K) < 1 ? 1 : 8 / (P * K), STEP = TOGETHER ? JOIN_WARPS : 1;
    __shared__ float factors[TOGETHER ? LINE_BLOCKS : 1], warps_max[JOIN_WARPS], warps_sum[JOIN_WARPS], others[TOGETHER ? JOIN_WARPS : 1][TOGETHER ? DP : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part0 = TOGETHER ? warp : 0;
    auto at = [&](int i, int r) { return part_row(line, job.c_first + i, i > 0 ? 0 : 1, r); };
    const float2* const ml = reinterpret_cast<const float2*>(line.part_ml);
    for (int base = TOGETHER ? r0 : r0 + warp * R; base < r1; base += TOGETHER ? 1 : JOIN_WARPS * R) {
        float v[R][P][K][V];
        auto request = [&](int i0) {
#pragma unroll
            for (int x = 0; x < R; ++x)
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const int part = i0 + i * STEP;
#pragma unroll
                        for (int e = 0; e < V; ++e) v[x][i][k][e] = 0.f;
                        if (part < job.parts && base + x < r1) piece_of<V>(v[x][i][k], line.part_o + at(part, base + x) * A.d, (lane + 32 * k) * V, A.d);
                    }
        };
        request(part0);
        float f[R], W[R];                          // of the lane's part (not TOGETHER); of the row
        if constexpr (TOGETHER) {
            float M = -INFINITY, mine = 0.f;
            for (int i = threadIdx.x; i < job.parts; i += THREADS) M = fmaxf(M, __ldcg(ml + at(i, base)).x);
            M = warp_max(M);
            if (lane == 0) warps_max[warp] = M;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < JOIN_WARPS; ++w) M = fmaxf(M, warps_max[w]);
            if (M == -INFINITY) M = 0.f;
            for (int i = threadIdx.x; i < job.parts; i += THREADS) {
                const float2 x = __ldcg(ml + at(i, base));
                const float e = expf(x.x - M);
                factors[i] = e;
                mine = fmaf(e, x.y, mine);
            }
            mine = warp_sum(mine);
            if (lane == 0) warps_sum[warp] = mine;
            __syncthreads();
            W[0] = 0.f;
#pragma unroll
            for (int w = 0; w < JOIN_WARPS; ++w) W[0] += warps_sum[w];
        } else {
#pragma unroll
            for (int x = 0; x < R; ++x) {
                const float2 mine = lane < job.parts && base + x < r1 ? __ldcg(ml + at(lane, base + x)) : make_float2(-INFINITY, 0.f);
                float M = warp_max(mine.x);
                if (M == -INFINITY) M = 0.f;
                f[x] = expf(mine.x - M);
                W[x] = warp_sum(f[x] * mine.y);
            }
        }
        float acc[R][K][V];
#pragma unroll
        for (int x = 0; x < R; ++x)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[x][k][e] = 0.f;
        for (int i0 = part0; i0 < job.parts; i0 += P * STEP) {
            if (i0 > part0) request(i0);
#pragma unroll
            for (int x = 0; x < R; ++x)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int part = i0 + i * STEP;
                    float fi;
                    if constexpr (TOGETHER) fi = part < job.parts ? factors[part] : 0.f;
                    else fi = __shfl_sync(0xffffffffu, f[x], part & 31);
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[x][k][e] = fmaf(fi, v[x][i][k][e], acc[x][k][e]);
                }
        }
        if constexpr (TOGETHER) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) others[warp][(lane + 32 * k) * V + e] = acc[0][k][e];
            __syncthreads();
        }
#pragma unroll
        for (int x = 0; x < R; ++x) {
            const int row = job.row0 + base + x;
            if (base + x >= r1) continue;
            const float inv = W[x] > 0.f || W[x] != W[x] ? 1.f / W[x] : 0.f;
            T* out = (T*)A.out + (size_t)(job.first + row / job.G) * A.out_stride + (size_t)(job.g * job.G + row % job.G) * A.d;
            if constexpr (TOGETHER) {
                for (int c = threadIdx.x; c < A.d; c += THREADS) {
                    float sum = 0.f;
#pragma unroll
                    for (int w = 0; w < JOIN_WARPS; ++w) sum += others[w][c];
                    out[c] = from_f32<T>(sum * inv);
                }
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if ((lane + 32 * k) * V + e < A.d) out[(lane + 32 * k) * V + e] = from_f32<T>(acc[x][k][e] * inv);
            }
        }
        if constexpr (TOGETHER) __syncthreads();   // what the next row writes has been read
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS)
tree_join_kernel(const TreeArgs A, const Line line) {
    pdl_launch_dependents();
    pdl_wait();
    const int* job_at = line.shared_jobs + blockIdx.x * 8;
    const JoinJob job{job_at[0], job_at[1], job_at[2], job_at[3], job_at[4], job_at[5], A.nh / A.nkv};
    if (job.parts < 2) return;
    const int mine = (int)blockIdx.x / 2 - job.c_first, r0 = job.rows * mine / job.parts, r1 = job.rows * (mine + 1) / job.parts;
    if (job.parts > JOIN_TOGETHER) join_rows<T, DP, 8, true>(A, line, job, r0, r1);
    else if (job.parts > 4) join_rows<T, DP, 8, false>(A, line, job, r0, r1);
    else if (job.parts > 2) join_rows<T, DP, 4, false>(A, line, job, r0, r1);
    else join_rows<T, DP, 2, false>(A, line, job, r0, r1);
}

long long scratch_floats(int d) { return line_floats(LINE_BLOCKS, RT, d, 0); }

template <typename T, int DP>
int launch_dp(const TreeArgs& A, const Line& line, cudaStream_t stream) {
    constexpr int smem = 4 * (RT * (DP + 4) + KT * (DP + 4) + KT * DP + RT * (KT + 4));
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(tree_attention_kernel<T, DP>, smem, &roomy)) return rc;
    const int rc = xb_launch(tree_attention_kernel<T, DP>, dim3(LINE_BLOCKS), dim3(THREADS), smem, stream, A, line);
    if (rc) return rc;
    return xb_launch(tree_join_kernel<T, DP>, dim3(2 * LINE_BLOCKS), dim3(THREADS), 0, stream, A, line);
}

template <typename T>
int launch(const TreeArgs& A, float* scratch, cudaStream_t stream) {
    Line line;
    line.two_from = A.tokens;
    // A tile a block while there are blocks enough: a tile takes 3 us of a block by itself, the join of its part half a microsecond.  One, two
    // and three tiles measured: 13.8, 18.7 and 21.0 us (8 nodes, 16 heads of 64 channels, 600 keys), 38.2, 38.2 and 48.0 (16 nodes, 4,096 keys).
    line.min_share = COST_ONE;
    line.row_mul = A.nh / A.nkv;
    line.row_div = RT;
    line.part_rows = RT;
    lay_out(line, LINE_BLOCKS, A.d, scratch);
    if (A.d <= 64) return launch_dp<T, 64>(A, line, stream);
    if (A.d <= 128) return launch_dp<T, 128>(A, line, stream);
    if (A.d <= 256) return launch_dp<T, 256>(A, line, stream);
    return launch_dp<T, 512>(A, line, stream);
}

}  // namespace

static int tree_attention(int dtype, void* out, const void* q, const void* k_new, const void* v_new, const void* k_cache, const void* v_cache,
                          const int* context, const int* token_start, const int* ancestors, const int* depth, const int* block_table,
                          long long out_stride, long long q_stride, long long k_stride, long long v_stride, int tokens, int requests, int words,
                          int table_stride, int nh, int nkv, int d, int page_size, int num_pages, int window, float scale, float* scratch,
                          int* err, cudaStream_t stream) {
    if (tokens <= 0 || requests <= 0) return 0;
    if (requests > LINE_REQUESTS || d < 1 || d > 512 || nkv < 1 || nh % nkv || page_size < 1 || (window > 0 && !depth)) return (int)cudaErrorInvalidValue;
    const TreeArgs A{out, q, k_new, v_new, k_cache, v_cache, context, token_start, ancestors, depth, block_table, out_stride, q_stride, k_stride, v_stride,
                     tokens, requests, words, table_stride, nh, nkv, d, page_size, num_pages, window, scale, err};
    if (!scratch || ((uintptr_t)scratch & 15)) return (int)cudaErrorInvalidValue;
    // the longest line that these shapes allow is counted in 32 bits
    const double jobs = (double)nkv * ((double)tokens * (nh / nkv) / RT + requests), tiles = (double)table_stride * page_size / KT + (double)tokens / KT + 2;
    if (jobs * (tiles * COST_TWO + COST_JOB) >= 2147483648.0) return (int)cudaErrorInvalidValue;
    if (dtype == XB_BF16 && tree_tc_takes(A)) return tree_tc_launch(A, scratch, stream);
    return dtype == XB_F32 ? launch<float>(A, scratch, stream) : launch<__nv_bfloat16>(A, scratch, stream);
}
XB_EXPORT int xb_tree_attention(const long long* words, int n) { return xb_by_words(tree_attention, words, n); }

// float32 numbers of scratch, on a 16-byte boundary, for a step of `tokens` drafted tokens: enough for either kernel
XB_EXPORT long long xb_tree_attention_scratch(int dtype, int tokens, int nh, int nkv, int d) {
    if (tokens <= 0 || nkv <= 0 || nh < nkv || d < 1) return 4;
    const long long any = scratch_floats(d), tc = dtype == XB_BF16 ? tree_tc_scratch(tokens, nh, nkv, d) : 0;
    return any > tc ? any : tc;
}
