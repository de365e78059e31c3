// Norms and rotation of a step's queries and keys, and its keys and values into pages of 4-bit codes (codes4.cuh), in one pass.
//
// Per token and head x of the projection's row [q heads | k heads | v heads]:  q and k: x * rsqrt(mean(x^2) + eps) * weight, then the
// first `rot` channels turned by the token's angle (pairs of neighbours, or of halves); queries go to rows of their own, keys and values to
// the token's slot, and on request to rows as the cache gives them back.
//
// Bound by its bytes in large steps, by a chain of trips (slot and position, angles, heads) in small ones.  8,192 tokens of 32 + 2 x 8 heads of 128
// channels in bfloat16, with the rows as the cache gives them back: 51 us, 216 MB, 4.2 TB/s; one token of 16 + 2 x 8 heads 2.5 us.
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

// Any head, rows on any boundary: a warp per (token, head), a group's channels one to a lane.  The 8,192 tokens above take 245 us this way, one token 4.3.
constexpr int ANY_WARPS = 8, ANY_MOST = 256;

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
        const uint32_t word = xb4::word_of(lo, hi);
        const float lift = xb4::scale_of(word) < xb4::TINY ? xb4::LIFT : 1.f, s = xb4::scale_of(word) * lift;
        const uint32_t code = __float_as_uint(xb4::raised_code(v * lift, s, xb4::least_of(word) * lift, xb4::reciprocal(s))) & 15u;
        if (values && c < d) values[c] = __float2bfloat16_rn(xb4::value_of(code, word));
        uint32_t eight = code << (4 * (lane & 7));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) eight |= __shfl_xor_sync(0xffffffffu, eight, o);
        if (!kept) continue;
        if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(page + ((long long)j * A.page_size + place) * xb4::GROUP_BYTES)[lane >> 3] = eight;
        if (lane == 0) reinterpret_cast<uint32_t*>(page + (long long)groups * A.page_size * xb4::GROUP_BYTES)[place * groups + j] = word;
    }
}

// Heads of a multiple of 8 channels, up to 256, whose rotation pairs whole vectors of 8 (halves of a multiple of 8) or neighbours: a lane has 8
// channels, LPH lanes a head, so a group's 32 channels are four lanes.  A warp takes one token and `each` times 32 / LPH of its heads, and keeps the
// token's angles.
constexpr int VEC_WARPS = 8;

__device__ __forceinline__ void load8(const float* x, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(x)[0], b = reinterpret_cast<const float4*>(x)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
// Eight numbers as they lie in memory.
template <typename T>
struct Eight {
    uint4 u[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Eight<T> fetch8(const T* x) {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(x)[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void numbers(const Eight<T>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint32_t w[4] = {r.u[i].x, r.u[i].y, r.u[i].z, r.u[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 2) v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            else v[4 * i + e] = __uint_as_float(w[e]);
        }
    }
}
__device__ __forceinline__ uint32_t pack2bf(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void store8(T* x, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(x) = make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7]));
    } else {
        reinterpret_cast<float4*>(x)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(x)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

constexpr int TURN_NONE = 0, TURN_HALVES = 1, TURN_PAIRS = 2;

template <typename T, int LPH, int TURN, bool FULL>
__global__ void __launch_bounds__(VEC_WARPS * 32, 4)
cache4_write_kernel(const WriteArgs A, int each) {
    constexpr int HEADS = 32 / LPH, AHEAD = 2;       // heads that are on their way
    pdl_overlap_few();
    const int lane = threadIdx.x & 31, li = lane & (LPH - 1), sub = lane / LPH, d = A.d;
    // a token's jobs: some for its query heads, then some for its keys and values
    const int q_jobs = (A.nh + HEADS * each - 1) / (HEADS * each), kv_jobs = (2 * A.nkv + HEADS * each - 1) / (HEADS * each);
    const unsigned job = blockIdx.x * VEC_WARPS + (threadIdx.x >> 5);
    const int t = (int)(job / (unsigned)(q_jobs + kv_jobs)), of_token = (int)(job % (unsigned)(q_jobs + kv_jobs));
    if (t >= A.tokens) return;
    const bool is_q = of_token < q_jobs, active = FULL || li * 8 < d;      // FULL: every lane has channels
    const int count = is_q ? A.nh : 2 * A.nkv, h0 = (is_q ? of_token : of_token - q_jobs) * HEADS * each + sub;
    const int c0 = active ? li * 8 : 0, groups = xb4::groups_of(d);
    const T* heads = static_cast<const T*>(A.qkv) + t * A.row_stride + c0 + (is_q ? 0 : (long long)A.nh * d);
    const int steps = min(each, (count - (h0 - sub) + HEADS - 1) / HEADS);
    Eight<T> next[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) next[j] = fetch8(heads + min(h0 + j * HEADS, count - 1) * d);
    // the token's angles: of the vector's pair in the other half (the sine with its sign), or of its own four pairs
    const int half = A.rot / 16;                   // vectors of a half
    const bool turns = TURN != TURN_NONE && active && c0 < A.rot, upper = TURN == TURN_HALVES && li >= half;
    const int other = (lane & ~(LPH - 1)) + (!turns ? li : (upper ? li - half : li + half));
    float cs[TURN == TURN_PAIRS ? 4 : 8], sn[TURN == TURN_PAIRS ? 4 : 8];
    const long long slot = A.slots[t];
    if constexpr (TURN != TURN_NONE) {
        const int at = A.positions[t];
        if (lane == 0 && slot >= 0 && (at < 0 || at >= A.max_pos)) atomicOr(A.err, XB_ERR_BAD_POSITION);
        const long long from = (long long)min(max(at, 0), A.max_pos - 1) * (A.rot / 2) + (!turns ? 0 : (TURN == TURN_PAIRS ? c0 / 2 : (upper ? c0 - half * 8 : c0)));
        if constexpr (TURN == TURN_PAIRS) {
            const float4 a = *reinterpret_cast<const float4*>(A.cos_t + from), b = *reinterpret_cast<const float4*>(A.sin_t + from);
            cs[0] = a.x, cs[1] = a.y, cs[2] = a.z, cs[3] = a.w, sn[0] = b.x, sn[1] = b.y, sn[2] = b.z, sn[3] = b.w;
        } else {
            load8(A.cos_t + from, cs);
            load8(A.sin_t + from, sn);
#pragma unroll
            for (int e = 0; e < 8; ++e) sn[e] = upper ? sn[e] : -sn[e];
        }
    }
    const float* w = is_q ? A.q_w : A.k_w;
    float wv[8];
    if (w) load8(w + c0, wv);
    const float one_over_d = 1.f / (float)d;
    // norm and rotation of a lane's channels (`wanted`: whether this head is normed and turned; the lanes of a warp exchange all the same)
    auto prepare = [&](float (&v)[8], bool wanted) {
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += active ? v[e] * v[e] : 0.f;
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, LPH);
            const float inv = rsqrtf(ss * one_over_d + A.eps);
            if (wanted) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * wv[e];
            }
        }
        if constexpr (TURN == TURN_PAIRS) {
            if (turns && wanted) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x0 = v[2 * e], x1 = v[2 * e + 1];
                    v[2 * e] = x0 * cs[e] - x1 * sn[e];
                    v[2 * e + 1] = x0 * sn[e] + x1 * cs[e];
                }
            }
        } else if constexpr (TURN == TURN_HALVES) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __shfl_sync(0xffffffffu, v[e], other);
            if (turns && wanted) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = fmaf(x[e], sn[e], v[e] * cs[e]);
            }
        }
    };
    if (is_q) {
        T* out = static_cast<T*>(A.q_out) + (long long)t * A.nh * d + c0;
#pragma unroll 1
        for (int i0 = 0; i0 < steps; i0 += AHEAD) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (i0 + j >= steps) break;
                const int h = h0 + (i0 + j) * HEADS;
                float v[8];
                numbers(next[j], v);
                if (i0 + AHEAD + j < steps) next[j] = fetch8(heads + min(h + AHEAD * HEADS, count - 1) * d);
                prepare(v, true);
                if (h < count && active) store8(out + h * d, v);
            }
        }
        return;
    }
    if (lane == 0 && slot >= A.num_slots) atomicOr(A.err, XB_ERR_BAD_PAGE);
    const bool kept = slot >= 0 && slot < A.num_slots;
    const int place = kept ? (int)(slot % A.page_size) : 0;
    const long long page_bytes = (long long)A.page_size * xb4::row_bytes(d), page = kept ? slot / A.page_size * A.nkv * page_bytes : 0;
    // where the lane's eight codes and its group's word go in a page; a lane behind the head writes the codes that fill its last group
    const int code_at = (int)((long long)(li >> 2) * A.page_size + place) * xb4::GROUP_BYTES + (li & 3) * 4, word_at = groups * A.page_size * xb4::GROUP_BYTES + (place * groups + (li >> 2)) * 4;
    const bool writes = kept && li < 4 * groups;
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
        const int h = h0 + i * HEADS;
        const bool is_k = h < A.nkv;
        float v[8];
        numbers(next[0], v);
#pragma unroll
        for (int j = 0; j + 1 < AHEAD; ++j) next[j] = next[j + 1];
        if (i + AHEAD < steps) next[AHEAD - 1] = fetch8(heads + min(h + AHEAD * HEADS, count - 1) * d);
        prepare(v, is_k);
        float lo = v[0], hi = v[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) lo = xb4::min_nan(lo, v[e]), hi = xb4::max_nan(hi, v[e]);
        if (!active) lo = INFINITY, hi = -INFINITY;        // (a last group may be shorter)
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = xb4::min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = xb4::max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const uint32_t word = xb4::word_of(lo, hi);
        const float s = xb4::scale_of(word), m = xb4::least_of(word);
        float of_s = s, of_m = m;
        if (s < xb4::TINY) {
            of_s *= xb4::LIFT, of_m *= xb4::LIFT;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= xb4::LIFT;
        }
        const float inv = xb4::reciprocal(of_s);
        uint32_t codes = 0u - 0x3f400000u;                     // (what the raised codes' upper bits come to, modulo 2^32)
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float c = xb4::raised_code(v[e], of_s, of_m, inv);
            codes += __float_as_uint(c) << (4 * e);
            y[e] = fmaf(s, c - xb4::CODE_UP, m);
        }
        if (h >= count) continue;
        const int g = is_k ? h : h - A.nkv;
        __nv_bfloat16* values = is_k ? A.k_values : A.v_values;
        if (values && active) store8(values + ((long long)t * A.nkv + g) * d + c0, y);
        uint8_t* to = (is_k ? A.k_cache : A.v_cache) + page + g * page_bytes;
        if (writes) *reinterpret_cast<uint32_t*>(to + code_at) = active ? codes : 0u;
        if (writes && (li & 3) == 0) *reinterpret_cast<uint32_t*>(to + word_at) = word;
    }
}

template <typename T, int LPH>
int launch_vec(const WriteArgs& A, cudaStream_t stream) {
    // As many heads a warp as leave every processor 32 warps, up to 16 times what lies side by side: a warp's angles and slot are a chain of trips.  8,192 tokens of
    // 32 + 2 x 8 heads with 4, 8 and 16: 78, 65 and 51 us.
    const int together = 32 / LPH;
    int each = 1;
    while (each < 16 && (long long)A.tokens * (A.nh + 2 * A.nkv) / (together * each * 2) >= 148 * 32) each *= 2;
    const long long jobs = (long long)A.tokens * ((A.nh + together * each - 1) / (together * each) + (2 * A.nkv + together * each - 1) / (together * each));
    auto go = [&](auto kernel) { return xb_launch_few(kernel, dim3((unsigned)((jobs + VEC_WARPS - 1) / VEC_WARPS)), dim3(VEC_WARPS * 32), 0, stream, A, each); };
    auto form = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        return !A.cos_t ? go(cache4_write_kernel<T, LPH, TURN_NONE, FULL>)
                        : (A.interleaved ? go(cache4_write_kernel<T, LPH, TURN_PAIRS, FULL>) : go(cache4_write_kernel<T, LPH, TURN_HALVES, FULL>));
    };
    return A.d == 8 * LPH ? form(std::true_type()) : form(std::false_type());
}

template <typename T>
bool vec_takes(const WriteArgs& A) {
    auto on16 = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    return A.d % 8 == 0 && A.d <= 256 && A.row_stride * sizeof(T) % 16 == 0 && on16(A.qkv) && on16(A.q_out) && on16(A.q_w) && on16(A.k_w) && on16(A.k_values) && on16(A.v_values) &&
           on16(A.cos_t) && on16(A.sin_t) && (!A.cos_t || A.rot % (A.interleaved ? 8 : 16) == 0);
}

template <typename T>
int launch(const WriteArgs& A, cudaStream_t stream) {
    if (vec_takes<T>(A)) {
        if (A.d <= 32) return launch_vec<T, 4>(A, stream);
        if (A.d <= 64) return launch_vec<T, 8>(A, stream);
        return A.d <= 128 ? launch_vec<T, 16>(A, stream) : launch_vec<T, 32>(A, stream);
    }
    const long long jobs = (long long)A.tokens * (A.nh + 2 * A.nkv);
    return xb_launch_few(cache4_write_any_kernel<T>, dim3((unsigned)((jobs + ANY_WARPS - 1) / ANY_WARPS)), dim3(ANY_WARPS * 32), 0, stream, A);
}

}  // namespace

static int cache4_write(int dtype, void* q_out, uint8_t* k_cache, uint8_t* v_cache, const void* qkv, const float* q_w, const float* k_w, const float* cos_t,
                        const float* sin_t, const int* positions, const long long* slots, __nv_bfloat16* k_values, __nv_bfloat16* v_values,
                        long long row_stride, long long num_slots, int tokens, int nh, int nkv, int d, int rot, int interleaved, int page_size, int max_pos,
                        float eps, int* err, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (d < 1 || d > ANY_MOST || nh < 0 || nkv < 1 || page_size < 1 || rot < 0 || rot > d || rot % 2 || (cos_t && max_pos < 1) || (long long)page_size * xb4::row_bytes(d) > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    if ((long long)tokens * (nh + 2 * nkv) > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    const WriteArgs A{q_out, k_cache, v_cache, qkv, q_w, k_w, rot ? cos_t : nullptr, sin_t, positions, slots, k_values, v_values, row_stride, num_slots, tokens, nh, nkv,
                      d, rot, interleaved, page_size, max_pos, eps, err};
    return dtype == XB_F32 ? launch<float>(A, stream) : launch<__nv_bfloat16>(A, stream);
}
XB_EXPORT int xb_cache4_write(const long long* words, int n) { return xb_by_words(cache4_write, words, n); }
