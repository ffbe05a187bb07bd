// Heads finished with positions of several axes (time, height, width): for every token of a fused projection's rows, queries and keys are
// normed (x / sqrt(mean x^2 + eps) * w, where weights are given), their pairs turned, pair i by the angle
//   positions[axis_of[i]][t] * inv_freq[i],
// values copied; queries go to q_out, keys and values into the paged caches at the token's slot (a negative one: a padded token, nothing is stored).
// The angle is a 64-bit product cut to a part of a turn: a 32-bit one is off by 2^-24 of the angle, 0.02 at position 300,000.  Cosine and sine are then
// sincospif of a number within half a turn; norm and rotation run in 32 bits and are rounded once.
// Bound by memory: every row is read and written once.  A block takes one token, all of its heads at once; a group of lanes takes a head, a lane two 16-byte
// vectors that the rotation pairs (half-split: u and u + half / VEC) or two of the head's vectors (pairs side by side), so no value changes lanes; the
// rows are asked for before the token's angles are worked out, once for all heads.
#define MB_LIB "rope_axes"
#define MB_LIB_ID 41
#include "common.cuh"
#include "launch.cuh"

#define AX_FEW 296                 // tokens a block each: up to two blocks an SM

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

// cos and sin of token t's angle of pair f.
__device__ __forceinline__ void token_angle(const AxesRows& p, int t, int f, float* cs, float* sn) {
    const int axis = min(max(p.axis_of[f], 0), p.axes - 1);
    const double turns = (double)p.positions[(size_t)axis * p.T + t] * (double)p.inv_freq[f] * 0.15915494309189533577;
    sincospif(2.0f * (float)(turns - rint(turns)), sn, cs);
}

// Where head `head` of token t goes, or null.
template <typename T>
__device__ __forceinline__ T* head_out(const AxesRows& p, int t, int head, int slot) {
    if (head < p.H) return (T*)p.q_out + ((size_t)t * p.H + head) * p.d;
    if (slot < 0 || slot >= p.cache_rows) return nullptr;
    const int kh = (head - p.H) % p.K;
    return (T*)(head < p.H + p.K ? p.k_cache : p.v_cache) + (((size_t)(slot / p.page_size) * p.K + kh) * p.page_size + (size_t)(slot % p.page_size)) * p.d;
}

template <typename T> struct Vec;
template <> struct Vec<bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& raw, float* v) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __bfloat1622float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        uint4 raw;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        return raw;
    }
};
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& raw, float* v) {
        v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* v) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
};

// LPG lanes a head (a power of two, at least the head's `units`), two vectors a lane, TT tokens a block.  Heads, halves and rows in whole 16-byte vectors.
template <typename T, int LPG, bool SIDE, int TT>
__global__ void __launch_bounds__(512) heads_axes_kernel(AxesRows p, int units) {
    constexpr int N = Vec<T>::N;
    extern __shared__ __align__(16) float ax_tab[];                 // [TT][half] cosines, [TT][half] sines
    const int t0 = blockIdx.x * TT, here = min(TT, p.T - t0), sub = threadIdx.x % LPG, group = threadIdx.x / LPG, groups = blockDim.x / LPG;
    const int vecs = p.d / N, turned = 2 * p.half / N;              // vectors of a head; the first `turned` of them turn
    // this lane's two vectors: the rotation's partners, or, of what does not turn (or turns inside a vector), the first and second half
    int va, vb;
    if (SIDE) { va = sub; vb = sub + units; }
    else if (sub < turned / 2) { va = sub; vb = sub + turned / 2; }
    else { va = turned + (sub - turned / 2); vb = va + (units - turned / 2); }
    const bool has_a = sub < units && va < vecs, has_b = sub < units && vb < vecs;
    PDL_ENTER();
    p.rows = pdl_fresh((const char*)p.rows); p.positions = pdl_fresh(p.positions); p.slots = pdl_fresh(p.slots);
    const T* row = (const T*)p.rows + (size_t)t0 * p.row_stride;
    float* cs = ax_tab;
    float* sn = ax_tab + TT * p.half;
    const bool turns = SIDE ? true : sub < turned / 2;
    const int rounds = (p.heads_total + groups - 1) / groups;       // the same for all lanes of a warp: the shuffles need them all
    for (int k = 0; k < rounds; ++k) {
        const int head = group + k * groups;
        const bool valid = head < p.heads_total;
        uint4 ra[TT], rb[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            ra[j] = rb[j] = make_uint4(0, 0, 0, 0);
            if (valid && j < here) {
                const T* at = row + (size_t)j * p.row_stride + (size_t)head * p.d;
                if (has_a) ra[j] = *reinterpret_cast<const uint4*>(at + va * N);
                if (has_b) rb[j] = *reinterpret_cast<const uint4*>(at + vb * N);
            }
        }
        if (k == 0 && p.half > 0) {                                 // (the rows are on their way)
            for (int i = threadIdx.x; i < here * p.half; i += blockDim.x) {
                const int j = i / p.half, f = i - j * p.half;
                token_angle(p, t0 + j, f, &cs[i], &sn[i]);
            }
            __syncthreads();
        }
        const float* w = head < p.H ? p.q_w : (head < p.H + p.K ? p.k_w : nullptr);
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            if (j >= here) break;
            float a[N], b[N];
            Vec<T>::unpack(ra[j], a);
            Vec<T>::unpack(rb[j], b);
            if (p.q_w != nullptr || p.k_w != nullptr) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < N; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
                for (int o = LPG / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w != nullptr) {
                    const float scale = 1.0f / sqrtf(ss / (float)p.d + p.eps);
                    if (has_a) {
#pragma unroll
                        for (int e = 0; e < N; ++e) a[e] = a[e] * scale * w[va * N + e];
                    }
                    if (has_b) {
#pragma unroll
                        for (int e = 0; e < N; ++e) b[e] = b[e] * scale * w[vb * N + e];
                    }
                }
            }
            if (head < p.H + p.K && p.half > 0) {
                const float *c = cs + j * p.half, *s = sn + j * p.half;
                if (SIDE) {
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        if (va < turned) {
                            const float x = a[2 * e], y = a[2 * e + 1], ce = c[va * (N / 2) + e], se = s[va * (N / 2) + e];
                            a[2 * e] = x * ce - y * se; a[2 * e + 1] = y * ce + x * se;
                        }
                        if (vb < turned) {
                            const float x = b[2 * e], y = b[2 * e + 1], ce = c[vb * (N / 2) + e], se = s[vb * (N / 2) + e];
                            b[2 * e] = x * ce - y * se; b[2 * e + 1] = y * ce + x * se;
                        }
                    }
                } else if (turns) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float x = a[e], y = b[e], ce = c[sub * N + e], se = s[sub * N + e];
                        a[e] = x * ce - y * se; b[e] = y * ce + x * se;
                    }
                }
            }
            if (valid) {
                T* dst = head_out<T>(p, t0 + j, head, head < p.H ? 0 : p.slots[t0 + j]);
                if (dst != nullptr) {
                    if (has_a) *reinterpret_cast<uint4*>(dst + va * N) = Vec<T>::pack(a);
                    if (has_b) *reinterpret_cast<uint4*>(dst + vb * N) = Vec<T>::pack(b);
                }
            }
        }
    }
}

// Any head size, rotary width and alignment: a warp takes a head through shared memory.
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
            const float scale = 1.0f / sqrtf(warp_sum(ss) / (float)p.d + p.eps);
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

template <typename T>
static int launch_axes(const AxesRows& p, cudaStream_t s) {
    constexpr int N = Vec<T>::N;
    const uintptr_t all = (uintptr_t)p.rows | (uintptr_t)p.q_out | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache;
    const bool whole = p.d % N == 0 && (all & 15) == 0 && p.row_stride % N == 0 && (p.interleaved ? (2 * p.half) % N == 0 : p.half % N == 0);
    const int vecs = p.d / N, turned = 2 * p.half / N;
    const int units = p.interleaved ? (vecs + 1) / 2 : turned / 2 + (vecs - turned + 1) / 2;
    if (whole && units <= 32) {
        int lpg = 4;
        while (lpg < units) lpg <<= 1;
        const int threads = min(512, (p.heads_total * lpg + 31) / 32 * 32);
        // many tokens: four a block, so that enough rows are on their way (8,007 tokens of 48 heads of 128: XX us, one a block 73); few: one, to have more blocks
        const int tt = p.T >= 4 * AX_FEW ? 4 : 1;
        const size_t smem = (size_t)max(1, 2 * tt * p.half) * sizeof(float);
        const dim3 grid((p.T + tt - 1) / tt);
#define AX_PICK(L, S) (tt == 4 ? launch_kernel(heads_axes_kernel<T, L, S, 4>, grid, dim3(threads), smem, s, 0, p, units) \
                               : launch_kernel(heads_axes_kernel<T, L, S, 1>, grid, dim3(threads), smem, s, 0, p, units))
#define AX_LAUNCH(L) (p.interleaved ? AX_PICK(L, true) : AX_PICK(L, false))
        if (lpg == 4) return AX_LAUNCH(4);
        if (lpg == 8) return AX_LAUNCH(8);
        if (lpg == 16) return AX_LAUNCH(16);
        return AX_LAUNCH(32);
#undef AX_LAUNCH
#undef AX_PICK
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
    const AxesRows p = {c->rows, const_cast<void*>(c->q_out), c->q_w, c->k_w, c->positions, c->axis_of, c->inv_freq, c->slots, c->write_kv ? const_cast<void*>(c->k_cache) : nullptr,
                        c->write_kv ? const_cast<void*>(c->v_cache) : nullptr, c->row_stride, c->cache_rows, c->eps, c->T, H, c->write_kv ? K : 0, d, c->axes, half, c->interleaved,
                        c->page_size, heads_total};
    if (c->dtype == MB_F32) return launch_axes<float>(p, s);
    if (c->dtype == MB_BF16) return launch_axes<bf16>(p, s);
    return MB_ERR_BAD_DTYPE;
}
