// Norms and rotation of a step's queries and keys, and its keys and values into pages of 4-bit codes (codes4.cuh), in one pass.
//
// Per token and head x of the projection's row [q heads | k heads | v heads]:  q and k: x * rsqrt(mean(x^2) + eps) * weight, then the
// first `rot` channels turned by the token's angle (pairs of neighbours, or of halves); queries go to rows of their own, keys and values to
// the token's slot, and on request to rows as the cache gives them back.
#include "codes4.cuh"

namespace {

struct WriteArgs {
    void* q_out;                   // [tokens, nh, d]
    uint8_t* k_cache;              // [pages, nkv, page_size * row_bytes(d)]
    uint8_t* v_cache;
    const void* qkv;               // [tokens, (nh + 2 nkv) d], rows `row_stride` elements apart
    const float* q_w;              // [d] or null: no norm
    const float* k_w;
    const float* cos_t;            // [max_pos, rot / 2] or null: no rotation
    const float* sin_t;
    const int* positions;          // [tokens]
    const long long* slots;        // [tokens]: page * page_size + place; -1: the token is not cached
    __nv_bfloat16* k_values;       // [tokens, nkv, d] or null
    __nv_bfloat16* v_values;
    long long row_stride, num_slots;
    int tokens, nh, nkv, d, rot, interleaved, page_size, max_pos;
    float eps;
    int* err;
};

// Where a token's codes of a group and its word lie in the page of a key/value head.
__device__ __forceinline__ uint8_t* page_of(const WriteArgs& A, uint8_t* cache, long long slot, int g) {
    return cache + (slot / A.page_size * A.nkv + g) * ((long long)A.page_size * xb4::row_bytes(A.d));
}

// Any head of up to 512 channels: a warp per (token, head), a group's channels one to a lane.
constexpr int ANY_WARPS = 8, ANY_MOST = 512;

template <typename T>
__global__ void __launch_bounds__(ANY_WARPS * 32)
cache4_write_any_kernel(const WriteArgs A) {
    __shared__ float turned[ANY_WARPS][ANY_MOST];
    pdl_overlap_few();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = A.nh + 2 * A.nkv;
    const long long job = (long long)blockIdx.x * ANY_WARPS + warp;
    if (job >= (long long)A.tokens * heads) return;
    const int t = (int)(job / heads), h = (int)(job % heads), d = A.d, groups = xb4::groups_of(d);
    const bool is_q = h < A.nh, is_k = !is_q && h < A.nh + A.nkv;
    const T* x = static_cast<const T*>(A.qkv) + t * A.row_stride + (long long)h * d;
    float* mine = turned[warp];
    float ss = 0.f;
    for (int c = lane; c < d; c += 32) {
        const float v = to_f32<T>(x[c]);
        mine[c] = v;
        ss += v * v;
    }
    ss = warp_sum(ss);
    const float* w = is_q ? A.q_w : (is_k ? A.k_w : nullptr);
    if (w) {
        const float inv = rsqrtf(ss / (float)d + A.eps);
        for (int c = lane; c < d; c += 32) mine[c] = mine[c] * inv * w[c];
    }
    __syncwarp();
    const long long slot = A.slots[t];
    if (A.cos_t && (is_q || is_k)) {
        const int at = A.positions[t], half = A.rot / 2;
        if ((at < 0 || at >= A.max_pos) && slot >= 0 && lane == 0) atomicOr(A.err, XB_ERR_BAD_POSITION);
        const long long row = (long long)min(max(at, 0), A.max_pos - 1) * half;      // (what is read instead lies in the table)
        for (int i = lane; i < half; i += 32) {
            const int a = A.interleaved ? 2 * i : i, b = A.interleaved ? 2 * i + 1 : i + half;
            const float c = A.cos_t[row + i], s = A.sin_t[row + i], x0 = mine[a], x1 = mine[b];
            mine[a] = x0 * c - x1 * s;
            mine[b] = x0 * s + x1 * c;
        }
        __syncwarp();
    }
    if (is_q) {
        T* out = static_cast<T*>(A.q_out) + ((long long)t * A.nh + h) * d;
        for (int c = lane; c < d; c += 32) out[c] = from_f32<T>(mine[c]);
        return;
    }
    const int g = is_k ? h - A.nh : h - A.nh - A.nkv;
    __nv_bfloat16* values = is_k ? A.k_values : A.v_values;
    if (values) values += ((long long)t * A.nkv + g) * d;
    bool kept = slot >= 0;
    if (kept && slot >= A.num_slots) {
        if (lane == 0) atomicOr(A.err, XB_ERR_BAD_PAGE);
        kept = false;
    }
    const int place = kept ? (int)(slot % A.page_size) : 0;
    uint8_t* page = page_of(A, is_k ? A.k_cache : A.v_cache, kept ? slot : 0, g);
    for (int j = 0; j < groups; ++j) {
        const int c = j * 32 + lane;
        const float v = mine[min(c, d - 1)];       // (lanes behind the head repeat its last channel, which changes no group's range)
        float lo = v, hi = v;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            lo = xb4::min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = xb4::max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const uint32_t word = xb4::word_of(lo, hi), code = xb4::code_of(v, word);
        if (values && c < d) values[c] = __float2bfloat16_rn(xb4::value_of(code, word));
        uint32_t eight = code << (4 * (lane & 7));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) eight |= __shfl_xor_sync(0xffffffffu, eight, o);
        if (!kept) continue;
        if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(page + ((long long)j * A.page_size + place) * xb4::GROUP_BYTES)[lane >> 3] = eight;
        if (lane == 0) reinterpret_cast<uint32_t*>(page + (long long)groups * A.page_size * xb4::GROUP_BYTES)[place * groups + j] = word;
    }
}

template <typename T>
int launch_any(const WriteArgs& A, cudaStream_t stream) {
    const long long jobs = (long long)A.tokens * (A.nh + 2 * A.nkv);
    return xb_launch_few(cache4_write_any_kernel<T>, dim3((unsigned)((jobs + ANY_WARPS - 1) / ANY_WARPS)), dim3(ANY_WARPS * 32), 0, stream, A);
}

}  // namespace

static int cache4_write(int dtype, void* q_out, uint8_t* k_cache, uint8_t* v_cache, const void* qkv, const float* q_w, const float* k_w, const float* cos_t,
                        const float* sin_t, const int* positions, const long long* slots, __nv_bfloat16* k_values, __nv_bfloat16* v_values,
                        long long row_stride, long long num_slots, int tokens, int nh, int nkv, int d, int rot, int interleaved, int page_size, int max_pos,
                        float eps, int* err, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (d < 1 || d > ANY_MOST || nh < 0 || nkv < 1 || page_size < 1 || rot < 0 || rot > d || rot % 2 || (cos_t && max_pos < 1)) return (int)cudaErrorInvalidValue;
    if ((long long)tokens * (nh + 2 * nkv) > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    const WriteArgs A{q_out, k_cache, v_cache, qkv, q_w, k_w, rot ? cos_t : nullptr, sin_t, positions, slots, k_values, v_values, row_stride, num_slots, tokens, nh, nkv,
                      d, rot, interleaved, page_size, max_pos, eps, err};
    return dtype == XB_F32 ? launch_any<float>(A, stream) : launch_any<__nv_bfloat16>(A, stream);
}
XB_EXPORT int xb_cache4_write(const long long* words, int n) { return xb_by_words(cache4_write, words, n); }
