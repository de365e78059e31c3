// What a step that verifies trees of drafted tokens does beside its model: the path that the model's own choices confirm, pages and
// slots for tokens whose number only the device knows, and the accepted tokens' keys and values into those slots.
#include "common.cuh"

namespace {

// ---- acceptance -------------------------------------------------------------------------------------------------------
// Request b has the nodes token_start[b] .. token_start[b + 1] - 1; parents[t] is a node's place in its own tree (the root's: -1;
// a parent comes before its children).  From the root on, the next node of the path is the child of lowest place whose token is
// targets[its parent], as long as there is one and the path has room.  A warp per request: 32 nodes are looked at with one read each and a
// vote.  Bound by the chain of trips, one for a node's target and one or two for its child: 1.5 us for a tree of 16 whose path is short, 4.6 us for
// 256 trees of 64 with paths of up to 12 (calls in a row; a launch by itself is 1.3).
__global__ void tree_accept_kernel(int* accepted, int* path, int* next_tokens, const int* drafted, const int* targets, const int* parents,
                                   const int* token_start, int requests, int tokens, int width) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, b = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 5);
    if (b >= requests) return;
    const int first = min(max(token_start[b], 0), tokens), n = min(max(token_start[b + 1], first), tokens) - first;
    int* mine = path + (size_t)b * width;
    int len = 0, at = n > 0 ? 0 : -1, last = -1;
    while (at >= 0 && len < width) {
        if (lane == 0) mine[len] = first + at;
        ++len;
        last = targets[first + at];
        int next = -1;
        for (int base = (at + 1) & ~31; base < n && next < 0; base += 32) {
            const int i = base + lane;
            const bool fits = i > at && i < n && parents[first + i] == at && drafted[first + i] == last;
            const unsigned who = __ballot_sync(0xffffffffu, fits);
            if (who) next = base + __ffs(who) - 1;
        }
        at = next;
    }
    for (int i = len + lane; i < width; i += 32) mine[i] = -1;
    if (lane == 0) {
        accepted[b] = len;
        next_tokens[b] = last;
    }
}

// ---- pages and slots -----------------------------------------------------------------------------------------------------
// Request b holds ceil(lengths[b] / page_size) pages, the first entries of its row of the block table, and gets new_tokens[b] more
// tokens; one that has ended (-1) gives its pages back.  Free pages lie in a ring of `ring_size` page ids, `ring[1]` of them from
// place ring[0] on: pages are taken at its head, in order of the requests, and given back at its end, so nothing that a block reads
// is written by another and the same call may be made twice.  A request whose pages are not all there gets none and no slots; its
// length stays.  Every block forms the requests' sums for itself and takes a share of the tokens: nothing waits for another block, and one
// launch does it.  Bound by trips (lengths, then a token's page): 5.0 us for 64 requests of 6 tokens, 5.5 us for 32 of 2,048 (1.9 MB written).
constexpr int SLOT_THREADS = 256;
constexpr int SLOT_REQUESTS = 8192;             // requests of a call: their starts lie in shared memory

struct SlotArgs {
    long long* slots;              // [capacity]: page * page_size + offset; -1: none
    int* positions;                // [capacity]
    int* request;                  // [capacity]: the token's request, -1 behind them all
    int* token_start;              // [requests + 1]
    int* lengths_out;              // [requests]
    int* ring_out;                 // head and count afterwards
    int* table;                    // [requests, table_stride]
    int* free_ring;                // [ring_size]
    const int* ring;               // head, count
    const int* lengths;            // [requests]
    const int* new_tokens;         // [requests]
    int requests, capacity, table_stride, page_size, ring_size;
    int* err;
};

struct Sums {
    long long tokens;              // (a request may ask for any number)
    int need, back;
};
__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return Sums{a.tokens + b.tokens, a.need + b.need, a.back + b.back}; }

// Exclusive prefix of `mine` over the block's threads; `total` receives the sum.
__device__ __forceinline__ Sums block_prefix(Sums mine, Sums* of_warps, Sums& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums v{__shfl_up_sync(0xffffffffu, incl.tokens, o), __shfl_up_sync(0xffffffffu, incl.need, o), __shfl_up_sync(0xffffffffu, incl.back, o)};
        if (lane >= o) incl = incl + v;
    }
    if (lane == 31) of_warps[warp] = incl;
    __syncthreads();
    Sums before{0, 0, 0};
    total = Sums{0, 0, 0};
    for (int w = 0; w < SLOT_THREADS / 32; ++w) {
        if (w < warp) before = before + of_warps[w];
        total = total + of_warps[w];
    }
    return Sums{before.tokens + incl.tokens - mine.tokens, before.need + incl.need - mine.need, before.back + incl.back - mine.back};
}

// The last of `n` runs that begins at or before x, of runs that begin at begin(0) = 0 <= begin(1) <= ...
template <typename Begin>
__device__ __forceinline__ int run_of(int x, int n, Begin begin) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (begin(mid) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(SLOT_THREADS)
cache_slots_kernel(const SlotArgs A) {
    extern __shared__ int starts[];                              // per request: tokens before it,
    int* need_before = starts + A.requests + 1;                  // pages taken before it (~ of them: it was not served),
    int* back_before = need_before + A.requests;                 // pages given back before it
    __shared__ Sums of_warps[SLOT_THREADS / 32];
    __shared__ int taken;
    pdl_launch_dependents();
    pdl_wait();
    const int each = (A.requests + SLOT_THREADS - 1) / SLOT_THREADS, b0 = (int)threadIdx.x * each, b1 = min(b0 + each, A.requests);
    const int ps = A.page_size, head = (A.ring[0] % A.ring_size + A.ring_size) % A.ring_size, count = min(max(A.ring[1], 0), A.ring_size);
    auto pages = [&](int len) { return (int)(((unsigned)len + (unsigned)(ps - 1)) / (unsigned)ps); };       // (the sum is below 2^32)
    // whether the request's pages, those it holds and those it asks for, fit its row of the table, and its length 32 bits; one whose do not
    // asks for none
    auto fits = [&](int len, int add) { return max(add, 0) <= 0x7fffffff - len && pages(len + max(add, 0)) <= A.table_stride; };
    auto sums_of = [&](int len, int add) {
        if (!fits(len, add)) return Sums{max(add, 0), 0, 0};
        if (add < 0) return Sums{0, 0, pages(len)};
        return Sums{add, pages(len + add) - pages(len), 0};
    };
    auto start_of = [](long long tokens) { return (int)min(tokens, 0x7fffffffLL); };
    Sums mine{0, 0, 0}, total;
    for (int b = b0; b < b1; ++b) mine = mine + sums_of(max(A.lengths[b], 0), A.new_tokens[b]);
    if (threadIdx.x == 0) taken = 0;
    Sums at = block_prefix(mine, of_warps, total);
    const bool first_block = blockIdx.x == 0;
    int most = 0;
    for (int b = b0; b < b1; ++b) {
        const int len = max(A.lengths[b], 0), add = A.new_tokens[b];
        const Sums s = sums_of(len, add);
        const bool served = fits(len, add) && (s.need == 0 || at.need + s.need <= count);
        starts[b] = start_of(at.tokens);
        need_before[b] = served ? at.need : ~at.need;
        back_before[b] = at.back;
        if (served && s.need > 0) most = at.need + s.need;
        if (first_block) {
            A.token_start[b] = start_of(at.tokens);
            A.lengths_out[b] = add < 0 ? 0 : (served ? len + add : len);
            if (!served) atomicOr(A.err, XB_ERR_NO_PAGE);
        }
        at = at + s;
    }
    if (most > 0) atomicMax(&taken, most);
    if (threadIdx.x == 0) starts[A.requests] = start_of(total.tokens);
    __syncthreads();
    const bool room = total.back + count <= A.ring_size;         // (more pages than the ring was made for: they are not taken back)
    if (first_block && threadIdx.x == 0) {
        A.token_start[A.requests] = start_of(total.tokens);
        A.ring_out[0] = (int)(((long long)head + taken) % A.ring_size);
        A.ring_out[1] = count - taken + (room ? total.back : 0);
        if (!room) atomicOr(A.err, XB_ERR_BAD_PAGE);
        if (total.tokens > A.capacity) atomicOr(A.err, XB_ERR_BAD_ROW);
    }
    auto ring_at = [&](int i) { return (int)(((long long)head + i) % A.ring_size); };
    auto needed = [&](int b) { return need_before[b] < 0 ? ~need_before[b] : need_before[b]; };
    const int threads = (int)gridDim.x * SLOT_THREADS, me = (int)blockIdx.x * SLOT_THREADS + (int)threadIdx.x;
    for (int i = me; i < min(taken, total.need); i += threads) { // new entries of the table: the i-th page from the ring's head
        const int b = run_of(i, A.requests, needed);
        if (need_before[b] >= 0) A.table[(size_t)b * A.table_stride + pages(max(A.lengths[b], 0)) + i - need_before[b]] = A.free_ring[ring_at(i)];
    }
    if (room)
        for (int i = me; i < total.back; i += threads) {         // pages that are given back
            const int b = run_of(i, A.requests, [&](int b) { return back_before[b]; });
            A.free_ring[ring_at(count + i)] = A.table[(size_t)b * A.table_stride + i - back_before[b]];
        }
    for (int t = me; t < A.capacity; t += threads) {
        if (t >= total.tokens) {
            A.slots[t] = -1;
            A.positions[t] = 0;
            A.request[t] = -1;
            continue;
        }
        const int b = run_of(t, A.requests, [&](int b) { return starts[b]; });
        const int len = max(A.lengths[b], 0), pos = len + min(t - starts[b], 0x7fffffff - len), place = pos / ps, held = pages(len);
        long long slot = -1;
        if (need_before[b] >= 0) {                               // (then its positions are all below its new length)
            const int page = place < held ? A.table[(size_t)b * A.table_stride + place] : A.free_ring[ring_at(need_before[b] + place - held)];
            if (page >= 0) slot = (long long)page * ps + pos % ps;
            else atomicOr(A.err, XB_ERR_BAD_PAGE);
        }
        A.slots[t] = slot;
        A.positions[t] = pos;
        A.request[t] = b;
    }
}

// ---- accepted rows into the cache ------------------------------------------------------------------------------------------
// Token i of the step (slots[i], the o-th new one of request b = request_of[i], o = i - token_start[b]) is drafted row path[b][o]:
// its keys and values of every layer go to its slot.  Grid (token, some layers); U: the unit of the copy, two bytes where a head's row is no
// multiple of 16.  A block finds its token's row and slot by four trips to memory, so it copies several layers where there are blocks
// enough, with four units a thread on their way.  Bound by memory and these trips: 452 accepted tokens in 36 layers (133 MB read and written) 25
// us, with a cold L2 33 (a copy of as many bytes takes 20); four in 28 layers 2.8 us.
constexpr int COMMIT_THREADS = 256, COMMIT_AHEAD = 4;
template <typename U>
__global__ void __launch_bounds__(COMMIT_THREADS)
cache_commit_kernel(const void* const* layers /* [layers][4]: k cache, v cache, new k, new v */, int num_layers, int layers_each, const long long* slots,
                    const int* request_of, const int* token_start, const int* path, int requests, int width, int rows, int nkv,
                    int units, int page_size, long long num_slots, int* err) {
    pdl_launch_dependents();
    pdl_wait();
    const int i = blockIdx.x;
    const int b = request_of[i];
    const long long slot = slots[i];
    if (b < 0 || b >= requests) return;
    const int o = i - token_start[b];
    if (slot < 0 || o < 0 || o >= width) return;
    const int row = path[(size_t)b * width + o];
    if (row < 0) return;
    if (row >= rows || slot >= num_slots) {
        if (threadIdx.x == 0) atomicOr(err, row >= rows ? XB_ERR_BAD_ROW : XB_ERR_BAD_PAGE);
        return;
    }
    const long long page = slot / page_size, off = slot % page_size;
    const int l0 = blockIdx.y * layers_each, l1 = min(l0 + layers_each, num_layers);
    for (int c = threadIdx.x; c < 2 * nkv * units; c += COMMIT_THREADS) {
        const int what = c / (nkv * units), g = c / units % nkv, u = c % units;
        const long long to = ((page * nkv + g) * page_size + off) * units + u, from = ((long long)row * nkv + g) * units + u;
        for (int l = l0; l < l1; l += COMMIT_AHEAD) {
            U v[COMMIT_AHEAD];
#pragma unroll
            for (int k = 0; k < COMMIT_AHEAD; ++k)
                if (l + k < l1) v[k] = ((const U*)layers[4 * (l + k) + 2 + what])[from];
#pragma unroll
            for (int k = 0; k < COMMIT_AHEAD; ++k)
                if (l + k < l1) ((U*)const_cast<void*>(layers[4 * (l + k) + what]))[to] = v[k];
        }
    }
}

}  // namespace

static int tree_accept(int* accepted, int* path, int* next_tokens, const int* drafted, const int* targets, const int* parents,
                       const int* token_start, int requests, int tokens, int width, cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (width < 1) return (int)cudaErrorInvalidValue;
    return xb_launch(tree_accept_kernel, dim3((requests + 3) / 4), dim3(128), 0, stream, accepted, path, next_tokens, drafted, targets, parents, token_start, requests,
                     tokens, width);
}
XB_EXPORT int xb_tree_accept(const long long* words, int n) { return xb_by_words(tree_accept, words, n); }

static int cache_slots(long long* slots, int* positions, int* request, int* token_start, int* lengths_out, int* ring_out, int* table, int* free_ring,
                       const int* ring, const int* lengths, const int* new_tokens, int requests, int capacity, int table_stride, int page_size,
                       int ring_size, int* err, cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (requests > SLOT_REQUESTS || page_size < 1 || ring_size < 1 || table_stride < 1 || (long long)requests * table_stride > 0x7fffffffLL)
        return (int)cudaErrorInvalidValue;
    const SlotArgs A{slots, positions, request, token_start, lengths_out, ring_out, table, free_ring, ring, lengths, new_tokens,
                     requests, capacity, table_stride, page_size, ring_size, err};
    int blocks = (capacity + SLOT_THREADS - 1) / SLOT_THREADS;
    blocks = blocks < 4 ? 4 : (blocks > 148 ? 148 : blocks);    // (four also where few tokens come: pages are given back beside them)
    const size_t smem = (3 * (size_t)requests + 1) * 4;         // (with the kernel's own arrays above the default from 4,084 requests on)
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(cache_slots_kernel, (3 * SLOT_REQUESTS + 1) * 4, &roomy)) return rc;
    return xb_launch(cache_slots_kernel, dim3(blocks), dim3(SLOT_THREADS), smem, stream, A);
}
XB_EXPORT int xb_cache_slots(const long long* words, int n) { return xb_by_words(cache_slots, words, n); }

static int cache_commit(const void* const* layers, int num_layers, const long long* slots, const int* request_of, const int* token_start,
                        const int* path, int tokens, int requests, int width, int rows, int nkv, int row_bytes, int page_size, long long num_slots,
                        int* err, cudaStream_t stream) {
    if (tokens <= 0 || num_layers <= 0 || requests <= 0) return 0;
    if (num_layers > 65535 || row_bytes < 2 || row_bytes % 2 || page_size < 1) return (int)cudaErrorInvalidValue;
    // Layers of a block: as many as leave four blocks a processor, up to 16.  One layer a block and this rule: 1,000 tokens of 24 layers (4 heads of
    // 64) 26.4 and 10.3 us, 452 of 36 (8 of 128) 28.0 and 25.4, 100 of 36 7.7 and 5.6, 30 of 28 in float32 7.1 and 5.1; eight blocks a processor: 6.3
    // and 6.9 for the last two, 24.8 for 452.
    const long long share = (long long)tokens * num_layers / (148 * 4);
    const int each = share < 1 ? 1 : (share > 16 ? 16 : (int)share);
    const dim3 grid(tokens, (num_layers + each - 1) / each);
    auto go = [&](auto kernel, int unit) {
        return xb_launch(kernel, grid, dim3(COMMIT_THREADS), 0, stream, layers, num_layers, each, slots, request_of, token_start, path, requests, width, rows, nkv,
                         row_bytes / unit, page_size, num_slots, err);
    };
    return row_bytes % 16 == 0 ? go(cache_commit_kernel<uint4>, 16) : go(cache_commit_kernel<uint16_t>, 2);
}
XB_EXPORT int xb_cache_commit(const long long* words, int n) { return xb_by_words(cache_commit, words, n); }
