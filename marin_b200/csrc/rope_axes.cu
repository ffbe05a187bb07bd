// Heads finished with positions of several axes (time, height, width): for every token of a fused projection's rows, queries and keys are
// normed (x / sqrt(mean x^2 + eps) * w, where weights are given), their pairs turned, pair i by the angle
//   positions[axis_of[i]][t] * inv_freq[i],
// values copied; queries go to q_out, keys and values into the paged caches at the token's slot (a negative one: a padded token, nothing is stored).
// The angle is a 64-bit product cut to a part of a turn: a 32-bit one is off by 2^-24 of the angle, 0.02 at position 300,000.  Cosine and sine are then
// sincospif of a number within half a turn; norm and rotation run in 32 bits and are rounded once.
// Bound by memory: every row is read and written once.  A group of lanes takes a head, a lane two 16-byte vectors that the rotation pairs (half-split: u and
// u + half / VEC) or two of the head's vectors (pairs side by side), so no value changes lanes.  Two blocks an SM take equal runs of tokens, all heads at once: weights stay
// in registers, three tokens' rows are on their way (a block a token had its threads wait for each token's rows and angles: 73 us at the first size below), and an angle is
// worked out once for all heads, a thread an angle, tokens ahead of its use (the 64-bit product and sincospif are as many instructions as a head's whole norm and rotation).
// Measured on B200: 8,007 tokens of 32 + 2 x 8 heads of 128, bfloat16, norm, three axes (197 MB): 37 us, 5.3 TB/s, 81 % of the copy rate (issue slots 64 % busy);
// 2,501 tokens of 16 + 2 x 16 heads of 80, float32, pairs side by side (77 MB): 17 us, 4.4 TB/s; eight tokens 3 us, a launch and two trips to memory.
#define MB_LIB "rope_axes"
#define MB_LIB_ID 41
#include "common.cuh"
#include "launch.cuh"
#include "mma_helpers.cuh"
#include "pair_math.cuh"

#ifndef AX_STAGES
#define AX_STAGES 3                // tokens whose rows are on their way
#endif
#define AX_SMS 148

struct AxesRows {
    const void* rows;              // [T] rows `row_stride` elements apart: H query heads, K key heads, K value heads of d
    void* q_out;                   // [T, H * d]
    const float* q_w;              // [d] or null
    const float* k_w;
    const int* positions;          // [axes, T]
    const int* axis_of;            // [rotary / 2]
    const float* inv_freq;         // [rotary / 2] or null: nothing turns
    const int* slots;              // [T]
    void* k_cache;                 // [pages][K][page_size][d]
    void* v_cache;
    long long row_stride, cache_rows;          // cache_rows: pages * page_size
    float eps;
    int T, H, K, d, axes, half, interleaved, page_size, heads_total;
};

// Sine and cosine of an angle given in turns.
__device__ __forceinline__ void turn_of(double turns, float* sn, float* cs) { sincospif(2.0f * (float)(turns - rint(turns)), sn, cs); }
// The same of token t's angle of pair f (1 / (2 pi) turns a radian).
__device__ __forceinline__ void token_angle(const AxesRows& p, int t, int f, float* cs, float* sn) {
    const int axis = min(max(p.axis_of[f], 0), p.axes - 1);
    turn_of((double)p.positions[(size_t)axis * p.T + t] * ((double)p.inv_freq[f] * 0.15915494309189533577), sn, cs);
}

// Where head `head` of token t goes, or null.
template <typename T>
__device__ __forceinline__ T* head_out(const AxesRows& p, int t, int head, int slot) {
    if (head < p.H) return (T*)p.q_out + ((size_t)t * p.H + head) * p.d;
    if (slot < 0 || slot >= p.cache_rows) return nullptr;
    const int kh = (head - p.H) % p.K;
    return (T*)(head < p.H + p.K ? p.k_cache : p.v_cache) + (((size_t)(slot / p.page_size) * p.K + kh) * p.page_size + (size_t)(slot % p.page_size)) * p.d;
}

// 16 bytes of a head as pairs of float32, and back (rounded to nearest).
template <typename T> struct Vec;
template <> struct Vec<bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& raw, uint64_t* v) {
        const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pair_of(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 pack(const uint64_t* v) {
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x, y;
            of_pair(v[i], x, y);
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r[i]) : "f"(y), "f"(x));
        }
        return make_uint4(r[0], r[1], r[2], r[3]);
    }
};
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& raw, uint64_t* v) {
        v[0] = pair_of(__uint_as_float(raw.x), __uint_as_float(raw.y));
        v[1] = pair_of(__uint_as_float(raw.z), __uint_as_float(raw.w));
    }
    static __device__ __forceinline__ uint4 pack(const uint64_t* v) {
        float x, y, z, w;
        of_pair(v[0], x, y);
        of_pair(v[1], z, w);
        return make_uint4(__float_as_uint(x), __float_as_uint(y), __float_as_uint(z), __float_as_uint(w));
    }
};
// N floats (at 16 bytes) as pairs; the same of half as many.
template <int N>
__device__ __forceinline__ void load_pairs(const float* from, uint64_t* v) {
    if (N == 2) { const float2 f = *reinterpret_cast<const float2*>(from); v[0] = pair_of(f.x, f.y); }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 f = reinterpret_cast<const float4*>(from)[i];
        v[2 * i] = pair_of(f.x, f.y);
        v[2 * i + 1] = pair_of(f.z, f.w);
    }
}
// Pairs side by side: (x, y) by the angle of each.
template <int N>
__device__ __forceinline__ void turn_inside(uint64_t* v, const float* c, const float* s) {
    uint64_t cc[N / 4 > 0 ? N / 4 : 1], ss[N / 4 > 0 ? N / 4 : 1];
    load_pairs<N / 2>(c, cc);
    load_pairs<N / 2>(s, ss);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        float x, y, ce[2], se[2];
        of_pair(v[i], x, y);
        of_pair(cc[i >> 1], ce[0], ce[1]);
        of_pair(ss[i >> 1], se[0], se[1]);
        v[i] = pair_of(x * ce[i & 1] - y * se[i & 1], y * ce[i & 1] + x * se[i & 1]);
    }
}

// LPG lanes a head (a power of two, at least the head's `units`), two vectors a lane.  Heads, halves and rows in whole 16-byte vectors.
// A block (x) takes `per_block` tokens one after the other, of the heads that its threads reach (y): the rows of the next AX_STAGES tokens are on their way
// (cp.async, every thread the vectors that it works on itself, so no barrier stands between), and the angles of the next `ng` tokens are worked out, one a
// thread, before those at hand are used.  A thread's head is the same throughout: its weights stay in registers, its addresses move by a row.
template <typename T, int LPG, bool SIDE>
__global__ void __launch_bounds__(512, 2) heads_axes_kernel(AxesRows p, int units, int ng, int per_block) {
    constexpr int N = Vec<T>::N;
    extern __shared__ __align__(16) uint8_t ax_smem[];
    const int threads = blockDim.x, tid = threadIdx.x, sub = tid % LPG, half = p.half;
    uint4* ring = reinterpret_cast<uint4*>(ax_smem) + tid;          // [stage][2][threads]
    float* angles = reinterpret_cast<float*>(ax_smem + (size_t)AX_STAGES * 2 * threads * 16);       // [2][ng][cosines, sines][half]
    long long* places = reinterpret_cast<long long*>(angles + 4 * ng * half);               // [2][ng]: the token's first element in a cache, or -1
    const int vecs = p.d / N, turned = 2 * half / N;                // vectors of a head; the first `turned` of them turn
    // this lane's two vectors: the rotation's partners, or, of what does not turn (or turns inside a vector), the first and second half
    int va, vb;
    if (SIDE) { va = sub; vb = sub + units; }
    else if (sub < turned / 2) { va = sub; vb = sub + turned / 2; }
    else { va = turned + (sub - turned / 2); vb = va + (units - turned / 2); }
    const int head = blockIdx.y * (threads / LPG) + tid / LPG;
    const bool valid = head < p.heads_total, has_a = valid && sub < units && va < vecs, has_b = valid && sub < units && vb < vecs;
    const bool is_q = head < p.H, is_k = !is_q && head < p.H + p.K;
    const bool turns_a = (is_q || is_k) && half > 0 && (SIDE ? va < turned : sub < turned / 2), turns_b = (is_q || is_k) && half > 0 && (SIDE ? vb < turned : sub < turned / 2);
    const int t0 = blockIdx.x * per_block, n = min(per_block, p.T - t0);
    PDL_ENTER();
    p.rows = pdl_fresh((const char*)p.rows); p.positions = pdl_fresh(p.positions); p.slots = pdl_fresh(p.slots);
    const T* from = (const T*)p.rows + (size_t)t0 * p.row_stride + (size_t)head * p.d;
    const T *from_a = from + va * N, *from_b = from + vb * N;
    int asked = 0, ask_stage = 0;
    auto fetch = [&]() {
        if (asked < n) {
            if (has_a) cp_async16(ring + ask_stage * 2 * threads, from_a);
            if (has_b) cp_async16(ring + (ask_stage * 2 + 1) * threads, from_b);
            from_a += p.row_stride; from_b += p.row_stride;
        }
        ++asked;
        ask_stage = ask_stage + 1 == AX_STAGES ? 0 : ask_stage + 1;
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < AX_STAGES; ++i) fetch();
    // angles and places of the tokens first .. first + ng - 1, into buffer `buf`
    const bool all_at_once = ng * half <= threads, one_each = all_at_once && tid < ng * half;
    const int my_token = half > 0 ? tid / half : 0, my_pair = half > 0 ? tid % half : 0;
    const int my_axis = one_each ? min(max(p.axis_of[my_pair], 0), p.axes - 1) : 0;
    const double my_freq = one_each ? (double)p.inv_freq[my_pair] * 0.15915494309189533577 : 0.0;
    const int* my_positions = p.positions + (size_t)my_axis * p.T + t0 + my_token;
    auto position_of = [&](int first) { return one_each && first + my_token < n ? my_positions[first] : 0; };
    auto prepare = [&](int first, int buf, int position) {
        if (first >= n) return;
        float* cs = angles + buf * 2 * ng * half;
        if (all_at_once) {
            if (one_each) turn_of((double)position * my_freq, &cs[(2 * my_token + 1) * half + my_pair], &cs[2 * my_token * half + my_pair]);
        } else {
            for (int i = tid; i < ng * half; i += threads)
                if (first + i / half < n) token_angle(p, t0 + first + i / half, i % half, &cs[2 * (i / half) * half + i % half], &cs[(2 * (i / half) + 1) * half + i % half]);
        }
        if (tid < ng) {
            const int slot = p.heads_total > p.H && first + tid < n ? p.slots[t0 + first + tid] : -1;
            places[buf * ng + tid] = slot >= 0 && slot < p.cache_rows ? ((long long)(slot / p.page_size) * p.K * p.page_size + slot % p.page_size) * p.d : -1;
        }
    };
    const float* w = is_q ? p.q_w : (is_k ? p.k_w : nullptr);
    const bool any_norm = p.q_w != nullptr || p.k_w != nullptr;
    const float inv_d = 1.0f / (float)p.d;
    uint64_t wa[N / 2], wb[N / 2];
    if (w != nullptr) {
        if (has_a) load_pairs<N>(w + va * N, wa);
        if (has_b) load_pairs<N>(w + vb * N, wb);
    }
    // where this thread's vectors go: a row of q_out a token, or from the token's place in a cache on
    T* to = is_q ? (T*)p.q_out + ((size_t)t0 * p.H + head) * p.d : (T*)(is_k ? p.k_cache : p.v_cache) + (size_t)(head - p.H - (is_k ? 0 : p.K)) * p.page_size * p.d;
    prepare(0, 0, position_of(0));
    int position = position_of(ng), stage = 0;
    for (int first = 0, buf = 0; first < n; first += ng, buf ^= 1) {
        __syncthreads();                                            // (this buffer's angles are there, and nobody reads the other's)
        prepare(first + ng, buf ^ 1, position);
        position = position_of(first + 2 * ng);
        const float* cs = angles + buf * 2 * ng * half;
        const int last = min(ng, n - first);
        for (int j = 0; j < last; ++j, cs += 2 * half) {
            cp_async_wait<AX_STAGES - 1>();
            uint64_t a[N / 2], b[N / 2];
            Vec<T>::unpack(has_a ? ring[stage * 2 * threads] : make_uint4(0, 0, 0, 0), a);
            Vec<T>::unpack(has_b ? ring[(stage * 2 + 1) * threads] : make_uint4(0, 0, 0, 0), b);
            stage = stage + 1 == AX_STAGES ? 0 : stage + 1;
            fetch();
            if (any_norm) {
                uint64_t sq = mul_pair(a[0], a[0]), sr = mul_pair(b[0], b[0]);
#pragma unroll
                for (int e = 1; e < N / 2; ++e) { sq = fma_pair(a[e], a[e], sq); sr = fma_pair(b[e], b[e], sr); }
                float s0, s1;
                of_pair(add_pair(sq, sr), s0, s1);
                float ss = s0 + s1;
#pragma unroll
                for (int o = LPG / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w != nullptr) {
                    const float scale = rsqrtf(fmaf(ss, inv_d, p.eps));
                    const uint64_t scales = pair_of(scale, scale);
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        a[e] = mul_pair(mul_pair(a[e], scales), wa[e]);
                        b[e] = mul_pair(mul_pair(b[e], scales), wb[e]);
                    }
                }
            }
            if (SIDE) {
                if (turns_a) turn_inside<N>(a, cs + va * (N / 2), cs + half + va * (N / 2));
                if (turns_b) turn_inside<N>(b, cs + vb * (N / 2), cs + half + vb * (N / 2));
            } else if (turns_a) {
                uint64_t cc[N / 2], ss[N / 2];
                load_pairs<N>(cs + sub * N, cc);
                load_pairs<N>(cs + half + sub * N, ss);
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const uint64_t x = a[e], y = b[e], minus = ss[e] ^ 0x8000000080000000ull;
                    a[e] = fma_pair(x, cc[e], mul_pair(y, minus));
                    b[e] = fma_pair(y, cc[e], mul_pair(x, ss[e]));
                }
            }
            const long long place = is_q ? 0 : places[buf * ng + j];
            if (place >= 0) {
                if (has_a) *reinterpret_cast<uint4*>(to + place + va * N) = Vec<T>::pack(a);
                if (has_b) *reinterpret_cast<uint4*>(to + place + vb * N) = Vec<T>::pack(b);
            }
            if (is_q) to += (size_t)p.H * p.d;
        }
    }
    cp_async_wait<0>();
}

// Any head size, rotary width and alignment: a warp takes a head through shared memory, four of a token's heads at a time, so a token's chain of trips bounds it: 16 + 2 x 16 heads of 80
// with 40 turning, bfloat16, halves apart, 8 tokens 17 us, 8,007 124 (3 and 33 by the kernel above with 80 turning).
template <typename T>
__global__ void __launch_bounds__(128) heads_axes_any_kernel(AxesRows p) {
    extern __shared__ float ax_tab[];
    float* cs = ax_tab;
    float* sn = ax_tab + p.half;
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* buf = ax_tab + 2 * p.half + (size_t)warp * p.d;
    PDL_ENTER();
    p.rows = pdl_fresh((const char*)p.rows); p.positions = pdl_fresh(p.positions); p.slots = pdl_fresh(p.slots);
    for (int f = threadIdx.x; f < p.half; f += blockDim.x) token_angle(p, t, f, &cs[f], &sn[f]);
    __syncthreads();
    const int slot = p.heads_total > p.H ? p.slots[t] : -1;
    for (int head = warp; head < p.heads_total; head += 4) {
        const T* src = (const T*)p.rows + (size_t)t * p.row_stride + (size_t)head * p.d;
        T* dst = head_out<T>(p, t, head, slot);
        if (dst == nullptr) continue;
        float ss = 0.0f;
        for (int i = lane; i < p.d; i += 32) { const float v = to_f32(src[i]); buf[i] = v; ss += v * v; }
        const float* w = head < p.H ? p.q_w : (head < p.H + p.K ? p.k_w : nullptr);
        if (w != nullptr) {
            const float scale = rsqrtf(warp_sum(ss) / (float)p.d + p.eps);
            for (int i = lane; i < p.d; i += 32) buf[i] = buf[i] * scale * w[i];
        }
        __syncwarp();
        if (head < p.H + p.K) {
            for (int i = lane; i < p.half; i += 32) {
                const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + p.half;
                const float x = buf[ia], y = buf[ib];
                buf[ia] = x * cs[i] - y * sn[i];
                buf[ib] = y * cs[i] + x * sn[i];
            }
            __syncwarp();
        }
        for (int i = lane; i < p.d; i += 32) dst[i] = from_f32<T>(buf[i]);
        __syncwarp();
    }
}

#define AX_SMEM_MOST (100 * 1024)
template <typename T, int LPG, bool SIDE>
static int ax_launch(dim3 grid, int threads, size_t smem, cudaStream_t s, const AxesRows& p, int units, int ng, int per_block) {
    static LaunchSmem allowed;
    const int rc = allowed.allow(heads_axes_kernel<T, LPG, SIDE>, AX_SMEM_MOST);
    if (rc != 0) return rc;
    return launch_kernel(heads_axes_kernel<T, LPG, SIDE>, grid, dim3(threads), smem, s, 0, p, units, ng, per_block);
}

template <typename T>
static int launch_axes(const AxesRows& p, cudaStream_t s) {
    constexpr int N = Vec<T>::N;
    const uintptr_t all = (uintptr_t)p.rows | (uintptr_t)p.q_out | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache;
    const bool whole = p.d % N == 0 && ((all | (uintptr_t)p.q_w | (uintptr_t)p.k_w) & 15) == 0 && p.row_stride % N == 0 && (p.interleaved ? (2 * p.half) % N == 0 : p.half % N == 0);
    const int vecs = p.d / N, turned = 2 * p.half / N;
    const int units = p.interleaved ? (vecs + 1) / 2 : turned / 2 + (vecs - turned + 1) / 2;
    if (whole && units <= 32 && p.half <= 1024) {
        int lpg = 4;
        while (lpg < units) lpg <<= 1;
        const int threads = min(512, (p.heads_total * lpg + 31) / 32 * 32);
        // Up to two blocks an SM, equal runs of tokens each; angles for as many tokens at once as a block has threads.
        const int reach = threads / lpg, parts = (p.heads_total + reach - 1) / reach, blocks = max(1, 2 * AX_SMS / parts);
        const int per_block = (p.T + blocks - 1) / blocks, ng = max(1, min(p.half > 0 ? threads / p.half : 8, per_block));
        const size_t smem = (size_t)AX_STAGES * 2 * threads * 16 + (size_t)4 * ng * p.half * sizeof(float) + (size_t)2 * ng * sizeof(long long);
        const dim3 grid((p.T + per_block - 1) / per_block, parts);
#define AX_LAUNCH(L) (p.interleaved ? ax_launch<T, L, true>(grid, threads, smem, s, p, units, ng, per_block) : ax_launch<T, L, false>(grid, threads, smem, s, p, units, ng, per_block))
        if (lpg == 4) return AX_LAUNCH(4);
        if (lpg == 8) return AX_LAUNCH(8);
        if (lpg == 16) return AX_LAUNCH(16);
        return AX_LAUNCH(32);
#undef AX_LAUNCH
    }
    const size_t smem = (size_t)(4 * p.d + 2 * p.half) * sizeof(float);
    if (smem > 48 * 1024) return MB_ERR_BAD_SIZE;
    return launch_kernel(heads_axes_any_kernel<T>, dim3(p.T), dim3(128), smem, s, 0, p);
}

// What a call hands over, in one piece (a caller in Python pays for every argument).
struct AxesCall {
    const void *rows, *q_out;
    const float *q_w, *k_w;
    const int *positions, *axis_of;
    const float* inv_freq;
    const int* slots;
    const void *k_cache, *v_cache;
    long long row_stride, cache_rows;
    float eps;
    int dtype, axes, rotary, interleaved, page_size, T, H, K, d, write_kv;
};

MB_API int mb_heads_axes(const AxesCall* c, cudaStream_t s) {
    if (c->T <= 0) return 0;
    const int half = c->inv_freq != nullptr ? c->rotary / 2 : 0, H = c->H, K = c->K, d = c->d;
    if (d <= 0 || H < 0 || K < 0 || c->rotary < 0 || c->rotary > d || (c->rotary & 1) || (half > 0 && c->axes <= 0) || (c->write_kv && (K <= 0 || c->page_size <= 0)) || H + K == 0)
        return MB_ERR_BAD_SIZE;
    const int heads_total = c->write_kv ? H + 2 * K : H;
    if (heads_total == 0) return 0;
    // queries may be finished where they lie (a thread, or a warp, reads a head before it writes it), but not over other rows
    const long long bytes = c->dtype == MB_F32 ? 4 : 2, row = (long long)H * d;
    const uintptr_t rows = (uintptr_t)c->rows, q_out = (uintptr_t)c->q_out;
    if (H > 0 && !(rows == q_out && c->row_stride == row) && rows < q_out + bytes * c->T * row && q_out < rows + bytes * ((c->T - 1) * c->row_stride + (long long)heads_total * d))
        return MB_ERR_BAD_SIZE;
    const AxesRows p = {c->rows, const_cast<void*>(c->q_out), c->q_w, c->k_w, c->positions, c->axis_of, c->inv_freq, c->slots, c->write_kv ? const_cast<void*>(c->k_cache) : nullptr,
                        c->write_kv ? const_cast<void*>(c->v_cache) : nullptr, c->row_stride, c->cache_rows, c->eps, c->T, H, c->write_kv ? K : 0, d, c->axes, half, c->interleaved,
                        c->page_size, heads_total};
    if (c->dtype == MB_F32) return launch_axes<float>(p, s);
    if (c->dtype == MB_BF16) return launch_axes<bf16>(p, s);
    return MB_ERR_BAD_DTYPE;
}
