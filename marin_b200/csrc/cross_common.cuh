// What the kernels of attention to an encoder's states share: their arguments, a row's range of positions, and a row's exact sums.
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G]   over lo_t <= j < min(hi_t, len_r),   0 where that range is empty;
// r is token t's request, len_r the length of its source, [lo_t, hi_t) its span (all positions without spans).  Keys and values lie in pages
// [page][kv head][position in page][d], looked up in the request's row of the block table.
// The rows that share a kv head's keys are (token, query head of the group) pairs, token by token: row i of a request is token i / G, head i % G.
#pragma once
#include "common.cuh"
#include "launch.cuh"

struct CrossArgs {
    const void* q;                 // [T] rows q_stride elements apart: H heads of d
    const void* k_cache;
    const void* v_cache;
    void* out;                     // [T, H * d]
    const int* block_table;        // [R, max_pages]
    const int* lens;               // [R]
    const int* cu_tokens;          // [R + 1]
    const int* spans;              // [T, 2] or null
    long long q_stride;
    int max_pages, K, G, d, page_shift;
    float scale;
};

// What a call hands over, in one piece (a caller in Python pays for every argument): requests first .. first + requests - 1 of a step of `tokens` tokens, none
// with more than max_query of them or a source longer than `longest`; chunks: how many blocks of a cluster share their keys (0: the launcher decides).
struct CrossCall {
    const void *q, *k_cache, *v_cache;
    void* out;
    const int *block_table, *lens, *cu_tokens, *spans;
    int* error_flag;
    long long q_stride, cache_pages;
    float scale;
    int dtype, max_pages, first, requests, max_query, tokens, chunks, longest, H, K, d, page_size;
};
static inline int page_shift_of(int page_size) {
    for (int b = 0; b < 24; ++b)
        if ((1 << b) == page_size) return b;
    return -1;
}
static inline CrossArgs cross_args(const CrossCall* c) {
    return {c->q, c->k_cache, c->v_cache, c->out, c->block_table, c->lens, c->cu_tokens, c->spans, c->q_stride, c->max_pages, c->K, c->H / c->K, c->d,
            page_shift_of(c->page_size), c->scale};
}
// What every kernel asks of a call: sizes that fit, a power of two of positions a page, results that do not lie over queries (which other blocks may still read).
static inline bool cross_call_fits(const CrossCall* c) {
    const int shift = page_shift_of(c->page_size);
    const long long bytes = c->dtype == MB_F32 ? 4 : 2;
    return shift >= 0 && c->K > 0 && c->K <= 65535 && c->H > 0 && c->H % c->K == 0 && c->d > 0 && c->max_pages >= 0 && ((long long)c->max_pages << shift) <= 0x7fffff00LL &&
           c->scale > 0.0f && c->q_stride >= 0 &&
           ((uintptr_t)c->q >= (uintptr_t)c->out + bytes * c->tokens * c->H * c->d || (uintptr_t)c->out >= (uintptr_t)c->q + bytes * ((c->tokens - 1) * c->q_stride + (long long)c->H * c->d));
}
static inline bool chunks_fit(int chunks) { return chunks == 1 || chunks == 2 || chunks == 4 || chunks == 8; }

// The positions token t of a request sees, cut to its source; (0, 0) where there are none.
__device__ __forceinline__ int2 cross_range(const CrossArgs& a, int t, int len) {
    int lo = 0, hi = len;
    if (a.spans != nullptr) { lo = max(0, a.spans[2 * (size_t)t]); hi = min(len, a.spans[2 * (size_t)t + 1]); }
    return hi > lo ? make_int2(lo, hi) : make_int2(0, 0);
}

// Which tile of which request a launch's place `x` is; (-1, 0): none.  Tiles of `size` rows.  All lanes of a warp call it.
// max_tiles > 0: all requests have so many of them (what the longest portion needs).  0: request r's begin at place floor(rows ahead of it / size) + r, which leaves each as
// many places as it needs and one at most over; found 32 requests at a time.  CROSS_SORTED (up to 32 requests): those of the longest sources come first, so that a launch
// whose blocks do not all fit at once ends with its short tiles.
#define CROSS_SORTED (-1)
__device__ __forceinline__ int2 cross_tile_of(const CrossArgs& a, int first, int requests, int rows_a_token, int size, int max_tiles, int x) {
    const int lane = threadIdx.x & 31;
    if (max_tiles == CROSS_SORTED) {
        const int r = first + min(lane, requests - 1), len = max(0, a.lens[r]), tokens = lane < requests ? a.cu_tokens[r + 1] - a.cu_tokens[r] : 0;
        const int tiles = (int)(((long long)tokens * rows_a_token + size - 1) / size);
        int ahead = 0;
        for (int i0 = 0; i0 < requests; i0 += 8)                     // (lanes past the last request have no tiles)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = i0 + e, other = __shfl_sync(0xffffffffu, len, i), theirs = __shfl_sync(0xffffffffu, tiles, i);
                if (other > len || (other == len && i < lane)) ahead += theirs;
            }
        const unsigned mine = __ballot_sync(0xffffffffu, x >= ahead && x < ahead + tiles);
        if (mine == 0) return make_int2(-1, 0);
        const int owner = __ffs(mine) - 1;
        return make_int2(first + owner, x - __shfl_sync(0xffffffffu, ahead, owner));
    }
    if (max_tiles > 0) return make_int2(first + x / max_tiles, x % max_tiles);
    const int base = a.cu_tokens[first];
    int lo = 0, n = requests, begins = 0;
    do {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const int place = lane * step < n ? (int)((long long)(a.cu_tokens[first + at] - base) * rows_a_token / size) + at : 0x7fffffff;
        const int k = max(0, __popc(__ballot_sync(0xffffffffu, place <= x)) - 1);
        begins = __shfl_sync(0xffffffffu, place, k);
        lo += k * step;
        n = min(step, n - k * step);
    } while (n > 1);
    return make_int2(first + lo, x - begins);
}
// The launch's blocks and max_tiles of it: by the longest portion where that leaves few blocks without rows (no search then), else by the rows there are.  (B200, bfloat16, 32
// heads of 128 over 8, the longest portion's tiles against the search: 31 requests of 16 tokens and one of 2,048 over 1,024 positions 129 and 64 us, 199 of 2 and one of 2,048
// over 500 646 and 192; in 32 bits, 16 heads of 64, 464 and 426, 656 and 569; portions of one length have the same blocks either way.  Six prompts of up to
// 507 tokens, 40 heads of 128 over 8, three spans each in sources of 0 to 2,250 positions: 54 us in the order of requests, the longest last, 41 with the longest first.)
struct CrossGrid { long long blocks; int max_tiles; };
static inline CrossGrid cross_grid(const CrossCall* c, int rows_a_token, int size) {
    const long long tiles = ((long long)c->max_query * rows_a_token + size - 1) / size, padded = tiles * c->requests, filled = c->requests + (long long)c->tokens * rows_a_token / size;
    const long long least = padded < filled ? padded : filled;
    if (c->requests > 1 && c->requests <= 32 && least * c->K > 2 * 148) return {least, CROSS_SORTED};
    if (padded <= filled + filled / 4) return {padded, (int)tiles};
    return {filled, 0};
}

template <typename T>
__device__ __forceinline__ const T* cross_row(const CrossArgs& a, const void* cache, const int* table, int kh, int key) {
    const size_t page = (size_t)table[key >> a.page_shift];
    return (const T*)cache + (((page * a.K + kh) << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * a.d;
}

// Four elements of a row of d from element c on, as they lie in memory (no branch between loads: many are on their way at once); what is past d is the row's last, to be left out by the
// caller.  WHOLE: d is a multiple of four and rows begin where four elements can be read at once (cross_whole).
template <typename T, bool WHOLE> struct CrossPiece;
template <> struct CrossPiece<float, true> {
    float4 raw;
    __device__ __forceinline__ void load(const float* row, int c, int d) { raw = *reinterpret_cast<const float4*>(row + min(c, d - 4)); }
    __device__ __forceinline__ float4 get() const { return raw; }
};
template <> struct CrossPiece<bf16, true> {
    uint2 raw;
    __device__ __forceinline__ void load(const bf16* row, int c, int d) { raw = *reinterpret_cast<const uint2*>(row + min(c, d - 4)); }
    __device__ __forceinline__ float4 get() const { return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u)); }
};
template <typename T> struct CrossPiece<T, false> {
    T raw[4];
    __device__ __forceinline__ void load(const T* row, int c, int d) {
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = row[min(c + e, d - 1)];
    }
    __device__ __forceinline__ float4 get() const { return make_float4(to_f32(raw[0]), to_f32(raw[1]), to_f32(raw[2]), to_f32(raw[3])); }
};
template <typename T>
__device__ __forceinline__ bool cross_whole(const CrossArgs& a) {
    return a.d % 4 == 0 && a.q_stride % 4 == 0 && (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & (4 * sizeof(T) - 1)) == 0;
}
__device__ __forceinline__ bool not_finite(float4 v) { return !(fabsf(v.x) <= 3.0e38f && fabsf(v.y) <= 3.0e38f && fabsf(v.z) <= 3.0e38f && fabsf(v.w) <= 3.0e38f); }

// In a tile whose rows see different positions a value that is not finite reaches all of them (0 * infinity).  A row's result that is not finite is right all the same where
//   * the row's own scores are not finite (its sum of weights, which are the row's alone, is NaN or 0: softmax gives NaN), or
//   * every value of the tile's positions that is not finite is one that the row sees.
// Else the row is worked out from its own range (cross_row_alone).  The call's other rows wait for that, so it is one pass over keys and values, a few positions at a time.
// (B200, bfloat16, 32 heads of 128 over 8, 512 tokens over 2,000 positions, 0.05 ms: 0.2 ms where all rows see a value that is NaN, 3.3 where every second row has to be worked
// out again, over 1,000 positions; 0.05 where a key is NaN.  64 tokens over 500 positions: 0.08 and 0.5; with a lane a position and every such row again 13.)
__device__ __forceinline__ bool cross_sum_speaks(float sum) { return sum > 0.0f && sum < INFINITY; }       // (false where the sum itself says that the result is NaN)

// The first and the last position of [from, to) with a value that is not finite, of one kv head; (0x7fffffff, -1): none.  P: pieces of four elements a lane (two for heads over
// 128).  All 32 lanes of a warp call it, and get the same.
template <typename T, int P, bool WHOLE>
__device__ __noinline__ int2 cross_odd_values(const CrossArgs& a, int kh, int request, int from, int to) {
    constexpr int U = 4;
    const int lane = threadIdx.x & 31;
    const int* table = a.block_table + (size_t)request * a.max_pages;
    int first = 0x7fffffff, last = -1;
    for (int key0 = from; key0 < to; key0 += U) {
        CrossPiece<T, WHOLE> v[U][P];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int p = 0; p < P; ++p) v[u][p].load(cross_row<T>(a, a.v_cache, table, kh, min(key0 + u, to - 1)), 4 * lane + 128 * p, a.d);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            bool odd = not_finite(v[u][0].get());
            if (P > 1) odd |= not_finite(v[u][P - 1].get());
            if (odd) { first = min(first, min(key0 + u, to - 1)); last = max(last, min(key0 + u, to - 1)); }
        }
    }
    return make_int2(__reduce_min_sync(0xffffffffu, first), __reduce_max_sync(0xffffffffu, last));
}
// Whether a row of this range has to be worked out again, `odd` being the tile's positions with values that are not finite.
__device__ __forceinline__ bool cross_not_its_own(int2 odd, int2 range) { return !(odd.y >= 0 && odd.x >= range.x && odd.y < range.y); }

// One row's result from its own range alone, by one warp, U positions at a time.  All 32 lanes call it.
template <typename T, int P, int U, bool WHOLE>
__device__ __noinline__ void cross_row_alone(const CrossArgs& a, int t, int head, int request, int2 range) {
    const int lane = threadIdx.x & 31, kh = head / a.G;
    const T* q = (const T*)a.q + (size_t)t * a.q_stride + (size_t)head * a.d;
    const int* table = a.block_table + (size_t)request * a.max_pages;
    const float sl2 = a.scale * 1.4426950408889634f;
    float4 qp[P], acc[P];
    bool in[P][4];                                                  // (elements past d: no part of a score)
#pragma unroll
    for (int p = 0; p < P; ++p) {
        CrossPiece<T, WHOLE> from;
        from.load(q, 4 * lane + 128 * p, a.d);
        qp[p] = from.get();
        acc[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) in[p][e] = 4 * lane + 128 * p + (WHOLE ? 0 : e) < a.d;
    }
    float m = -INFINITY, l = 0.0f;
    for (int key0 = range.x; key0 < range.y; key0 += U) {
        CrossPiece<T, WHOLE> k[U][P], v[U][P];
#pragma unroll
        for (int u = 0; u < U; ++u) {                               // (past the range: its last position, without a weight)
            const int key = min(key0 + u, range.y - 1);
            const T *keys = cross_row<T>(a, a.k_cache, table, kh, key), *values = cross_row<T>(a, a.v_cache, table, kh, key);
#pragma unroll
            for (int p = 0; p < P; ++p) { k[u][p].load(keys, 4 * lane + 128 * p, a.d); v[u][p].load(values, 4 * lane + 128 * p, a.d); }
        }
        float s[U], top = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 kp = k[u][p].get();
                s[u] += (in[p][0] ? qp[p].x * kp.x : 0.0f) + (in[p][1] ? qp[p].y * kp.y : 0.0f) + ((in[p][2] ? qp[p].z * kp.z : 0.0f) + (in[p][3] ? qp[p].w * kp.w : 0.0f));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) { s[u] = warp_sum(s[u]) * sl2; top = fmaxf(top, s[u]); }
        const float base = top == -INFINITY ? 0.0f : top, corr = exp2f(m - base);
        m = top;
        l *= corr;
#pragma unroll
        for (int p = 0; p < P; ++p) { acc[p].x *= corr; acc[p].y *= corr; acc[p].z *= corr; acc[p].w *= corr; }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (key0 + u >= range.y) continue;
            const float w = exp2f(s[u] - base);
            l += w;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float4 vp = v[u][p].get();
                acc[p].x = fmaf(w, vp.x, acc[p].x); acc[p].y = fmaf(w, vp.y, acc[p].y); acc[p].z = fmaf(w, vp.z, acc[p].z); acc[p].w = fmaf(w, vp.w, acc[p].w);
            }
        }
    }
    T* out = (T*)a.out + ((size_t)t * a.K * a.G + head) * a.d;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = 4 * lane + 128 * p;
        const float of[4] = {acc[p].x, acc[p].y, acc[p].z, acc[p].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < a.d) out[c + e] = from_f32<T>(range.y > range.x ? of[e] / l : 0.0f);
    }
}

// A float from the shared memory of CTA `rank` of this cluster, at the address `addr` has in this CTA.
__device__ __forceinline__ float cross_peer(uint32_t addr, int rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ float4 cross_peer4(uint32_t addr, int rank) {
    uint32_t remote;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
    return v;
}
// One row's partial results of `blocks` (up to 32) blocks of a cluster: lane c asks block c for its maximum and sum; back come that block's factor (lane c) and the sum.
// EXACT: exp2f, else the special-function unit's.
template <bool EXACT>
__device__ __forceinline__ float cross_factor(const float* m, const float* l, int blocks, float& sum) {
    const int lane = threadIdx.x & 31;
    const float mine = lane < blocks ? cross_peer((uint32_t)__cvta_generic_to_shared(m), lane) : -INFINITY;
    const float part = lane < blocks ? cross_peer((uint32_t)__cvta_generic_to_shared(l), lane) : 0.0f;
    const float top = warp_max(mine), x = mine - (top == -INFINITY ? 0.0f : top);
    float f;
    if (EXACT) f = exp2f(x);
    else asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(x));
    sum = warp_sum(lane < blocks ? f * part : 0.0f);
    return f;
}
// Four columns of the row (from `o` on) added over the blocks in rank order, each times its factor.
__device__ __forceinline__ float4 cross_join4(const float* o, float factor, int blocks) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = 0; c < blocks; ++c) {
        const float w = __shfl_sync(0xffffffffu, factor, c);
        const float4 p = cross_peer4((uint32_t)__cvta_generic_to_shared(o), c);
        v.x = fmaf(w, p.x, v.x); v.y = fmaf(w, p.y, v.y); v.z = fmaf(w, p.z, v.z); v.w = fmaf(w, p.w, v.w);
    }
    return v;
}
__device__ __forceinline__ void cross_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
