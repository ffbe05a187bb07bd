// Attention to an encoder's states in 32-bit arithmetic on the CUDA cores: float32 inputs, and bfloat16 ones of the layouts that the tensor-core
// kernels do not take (the formula and the layout of rows: cross_common.cuh).
// A block takes BM rows (token, head of the group) of one request and kv head and walks its keys in tiles of 64 with a running maximum and sum:
//   S [BM x 64] = Q K^T    each thread BM / 16 rows x 4 keys, four elements of d a step from shared memory;
//   P = exp2(S - m)        rows over 16 lanes; P through shared memory;
//   O [BM x d] += P V      each thread BM / 16 rows x d / 16 columns, in registers.
// A tile's values are asked for (cp.async) before S, the next tile's keys before the softmax.
// Work split: the source is cut into up to eight chunks by its own length alone, a cluster's blocks take one each and add their partial results in
// shared memory in chunk order.  A row's arithmetic depends on its request's source and its range only, not on the batch, the portion or BM: the same bits.
// Bound by multiply-adds (portions: two of them a (row, key, element of d)) or by the latency of the tiles (few rows).
#define MB_LIB "attention_cross"
#define MB_LIB_ID 42
#include "cross_common.cuh"

#define CX_BN 64
#define CX_CHUNK 256               // keys a chunk at least: below that a block's tiles cost less than the cluster's meeting
#define CX_CHUNKS 8
#define CX_PSTRIDE (CX_BN + 4)

__host__ __device__ __forceinline__ int cross_chunks(int len) {
    int c = 1;
    while (c < CX_CHUNKS && c * CX_CHUNK < len) c <<= 1;
    return c;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 64 keys' (or values') rows of one kv head as float32, rows LD apart; positions outside [lo, hi) and columns past d are zeros.
template <typename T, int LD>
__device__ __forceinline__ void cross_tile(float* dst, const CrossArgs& a, const void* cache, const int* table, int kh, int key0, int lo, int hi, bool whole) {
    constexpr int PIECES = (LD - 4) / 4;
    for (int i = threadIdx.x; i < CX_BN * PIECES; i += 256) {
        const int row = i / PIECES, c = (i % PIECES) * 4, key = key0 + row;
        float* to = dst + row * LD + c;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (key >= lo && key < hi && c < a.d) {
            const T* from = cross_row<T>(a, cache, table, kh, key) + c;
            if (sizeof(T) == 4 && whole) { cp_async16(to, from); continue; }
            v.x = to_f32(from[0]);
            if (c + 1 < a.d) v.y = to_f32(from[1]);
            if (c + 2 < a.d) v.z = to_f32(from[2]);
            if (c + 3 < a.d) v.w = to_f32(from[3]);
        }
        *reinterpret_cast<float4*>(to) = v;
    }
    cp_async_commit();
}

template <typename T, int BM, int DCH>
__global__ void __launch_bounds__(256) attention_cross_kernel(const __grid_constant__ CrossArgs arg, int first_request, int max_tiles, int whole) {
    constexpr int RM = BM / 16, LD = DCH * 64 + 4;
    extern __shared__ __align__(16) float cx_smem[];
    float* sQ = cx_smem;                                            // [BM][LD]; later the partial results
    float* sK = sQ + BM * LD;
    float* sV = sK + CX_BN * LD;
    float* sP = sV + CX_BN * LD;                                    // [BM][CX_PSTRIDE]
    __shared__ float s_m[BM], s_l[BM];
    __shared__ int s_lo[BM], s_hi[BM], s_first, s_last;
    PDL_ENTER();
    CrossArgs a = arg;
    a.q = pdl_fresh((const char*)a.q); a.k_cache = pdl_fresh((const char*)a.k_cache); a.v_cache = pdl_fresh((const char*)a.v_cache);
    a.block_table = pdl_fresh(a.block_table); a.lens = pdl_fresh(a.lens); a.cu_tokens = pdl_fresh(a.cu_tokens); a.spans = pdl_fresh(a.spans);
    const int r = first_request + blockIdx.x / max_tiles, tile = blockIdx.x % max_tiles, kh = blockIdx.y;
    const int rank = blockIdx.z, t0 = a.cu_tokens[r], rows = (a.cu_tokens[r + 1] - t0) * a.G, row0 = tile * BM;
    if (row0 >= rows) return;                                       // (all blocks of a cluster)
    const int len = max(0, min(a.lens[r], a.max_pages << a.page_shift));
    const int chunks = min(cross_chunks(len), (int)gridDim.z), H = a.K * a.G;
    const int* table = a.block_table + (size_t)r * a.max_pages;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    if (tid == 0) { s_first = len; s_last = 0; }
    __syncthreads();
    if (tid < BM) {
        int2 range = make_int2(0, 0);
        if (row0 + tid < rows) range = cross_range(a, t0 + (row0 + tid) / a.G, len);
        s_lo[tid] = range.x; s_hi[tid] = range.y;
        if (range.y > range.x) { atomicMin(&s_first, range.x); atomicMax(&s_last, range.y); }
    }
    for (int i = tid; i < BM * LD; i += 256) {
        const int row = i / LD, c = i % LD;
        float v = 0.0f;
        if (row0 + row < rows && c < a.d) {
            const int at = row0 + row;
            v = to_f32(((const T*)a.q)[(size_t)(t0 + at / a.G) * a.q_stride + (size_t)(kh * a.G + at % a.G) * a.d + c]);
        }
        sQ[i] = v;
    }
    __syncthreads();
    const int tiles = (len + CX_BN - 1) / CX_BN, per = (tiles + chunks - 1) / chunks;
    const int from = max(rank * per, s_first / CX_BN);
    const int to = rank < chunks && s_last > s_first ? min(min(tiles, (rank + 1) * per), (s_last + CX_BN - 1) / CX_BN) : 0;
    const float sl2 = a.scale * 1.4426950408889634f;
    float m[RM], l[RM], o[RM][DCH][4];
    int lo[RM], hi[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        m[i] = -INFINITY; l[i] = 0.0f;
        lo[i] = s_lo[ty * RM + i]; hi[i] = s_hi[ty * RM + i];
#pragma unroll
        for (int c = 0; c < DCH; ++c) o[i][c][0] = o[i][c][1] = o[i][c][2] = o[i][c][3] = 0.0f;
    }
    const int first = s_first, last = s_last, steps = (a.d + 3) / 4;
    if (from < to) cross_tile<T, LD>(sK, a, a.k_cache, table, kh, from * CX_BN, first, last, whole);
    for (int kt = from; kt < to; ++kt) {
        const int key0 = kt * CX_BN;
        cross_tile<T, LD>(sV, a, a.v_cache, table, kh, key0, first, last, whole);
        cp_async_wait<1>();
        __syncthreads();
        float s[RM][4];
#pragma unroll
        for (int i = 0; i < RM; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll 2
        for (int x = 0; x < steps; ++x) {
            float4 kv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * LD + 4 * x);
#pragma unroll
            for (int i = 0; i < RM; ++i) {
                const float4 qv = *reinterpret_cast<const float4*>(sQ + (ty * RM + i) * LD + 4 * x);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(qv.x, kv[j].x, s[i][j]);
                    s[i][j] = fmaf(qv.y, kv[j].y, s[i][j]);
                    s[i][j] = fmaf(qv.z, kv[j].z, s[i][j]);
                    s[i][j] = fmaf(qv.w, kv[j].w, s[i][j]);
                }
            }
        }
        __syncthreads();
        if (kt + 1 < to) cross_tile<T, LD>(sK, a, a.k_cache, table, kh, key0 + CX_BN, first, last, whole);
        else cp_async_commit();
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = key0 + tx + 16 * j;
                s[i][j] = key >= lo[i] && key < hi[i] ? s[i][j] * sl2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float m_new = fmaxf(m[i], mx), base = m_new == -INFINITY ? 0.0f : m_new, corr = exp2f(m[i] - base);
            m[i] = m_new;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float pj = exp2f(s[i][j] - base);
                sum += pj;
                sP[(ty * RM + i) * CX_PSTRIDE + tx + 16 * j] = pj;
            }
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            l[i] = l[i] * corr + sum;
#pragma unroll
            for (int c = 0; c < DCH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][c][e] *= corr;
        }
        cp_async_wait<1>();
        __syncthreads();
#pragma unroll 2
        for (int j = 0; j < CX_BN; j += 4) {
            float4 pv[RM];
#pragma unroll
            for (int i = 0; i < RM; ++i) pv[i] = *reinterpret_cast<const float4*>(sP + (ty * RM + i) * CX_PSTRIDE + j);
#pragma unroll
            for (int c = 0; c < DCH; ++c) {
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const float4 v = *reinterpret_cast<const float4*>(sV + (j + jj) * LD + c * 64 + tx * 4);
#pragma unroll
                    for (int i = 0; i < RM; ++i) {
                        const float w = jj == 0 ? pv[i].x : jj == 1 ? pv[i].y : jj == 2 ? pv[i].z : pv[i].w;
                        o[i][c][0] = fmaf(w, v.x, o[i][c][0]);
                        o[i][c][1] = fmaf(w, v.y, o[i][c][1]);
                        o[i][c][2] = fmaf(w, v.z, o[i][c][2]);
                        o[i][c][3] = fmaf(w, v.w, o[i][c][3]);
                    }
                }
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int row = ty * RM + i;
        if (tx == 0) { s_m[row] = m[i]; s_l[row] = l[i]; }
#pragma unroll
        for (int c = 0; c < DCH; ++c) *reinterpret_cast<float4*>(sQ + row * LD + c * 64 + tx * 4) = make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
    }
    if (gridDim.z > 1) cross_cluster_sync(); else __syncthreads();
    // block `rank` finishes rows rank, rank + gridDim.z, ...: a warp a row, the chunks in their order
    const int warp = tid >> 5, lane = tid & 31;
    for (int row = rank + warp * (int)gridDim.z; row < BM; row += 8 * (int)gridDim.z) {
        if (row0 + row >= rows) break;
        const bool sees = s_hi[row] > s_lo[row];
        float sum = s_l[row], factor = 1.0f;
        if (gridDim.z > 1) factor = cross_factor<true>(&s_m[row], &s_l[row], chunks, sum);
        const int t = t0 + (row0 + row) / a.G, head = kh * a.G + (row0 + row) % a.G;
        T* out = (T*)a.out + ((size_t)t * H + head) * a.d;
        bool odd = false;
        for (int c0 = 0; c0 < a.d; c0 += 128) {
            const int c = c0 + 4 * lane;
            const float* from = sQ + row * LD + min(c, LD - 4);
            float4 v = gridDim.z > 1 ? cross_join4(from, factor, chunks) : *reinterpret_cast<const float4*>(from);
            v = sees ? make_float4(v.x / sum, v.y / sum, v.z / sum, v.w / sum) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            odd |= c < a.d && not_finite(v);
            if (c < a.d) out[c] = from_f32<T>(v.x);
            if (c + 1 < a.d) out[c + 1] = from_f32<T>(v.y);
            if (c + 2 < a.d) out[c + 2] = from_f32<T>(v.z);
            if (c + 3 < a.d) out[c + 3] = from_f32<T>(v.w);
        }
        if (a.spans != nullptr && __any_sync(0xffffffffu, odd)) { __syncwarp(); cross_row_alone<T>(arg, t, head, r, make_int2(s_lo[row], s_hi[row])); }
    }
    if (gridDim.z > 1) cross_cluster_sync();                        // (a block's shared memory is read until here)
}

template <typename T, int BM, int DCH>
static int launch_cross(const CrossArgs& a, int first_request, int requests, int max_tiles, int clusters, int whole, cudaStream_t s) {
    constexpr int LD = DCH * 64 + 4;
    const size_t smem = ((size_t)(BM + 2 * CX_BN) * LD + BM * CX_PSTRIDE) * sizeof(float);
    static LaunchSmem allowed;
    const int rc = allowed.allow(attention_cross_kernel<T, BM, DCH>, smem);
    if (rc != 0) return rc;
    return launch_kernel(attention_cross_kernel<T, BM, DCH>, dim3((unsigned)(requests * max_tiles), a.K, clusters), dim3(256), smem, s, clusters, a, first_request,
                         max_tiles, whole);
}

MB_API int mb_attention_cross(const CrossCall* c, cudaStream_t s) {
    if (c->requests <= 0 || c->max_query <= 0) return 0;
    if (!cross_call_fits(c) || c->d > 256) return MB_ERR_BAD_SIZE;
    const CrossArgs a = cross_args(c);
    const int whole = c->dtype == MB_F32 && a.d % 4 == 0 && (((uintptr_t)c->k_cache | (uintptr_t)c->v_cache) & 15) == 0;
    // up to 16 rows (single tokens): tiles of 16, a quarter of the multiply-adds that a tile of 64 would spend on rows that are not there
    const long long rows = (long long)c->max_query * a.G;
    const int bm = rows <= 16 ? 16 : 64;
    const long long tiles = (rows + bm - 1) / bm;
    if (tiles * c->requests > 0x7fffffffLL) return MB_ERR_BAD_SIZE;
    const int clusters = cross_chunks(c->longest), dch = (a.d + 63) / 64;
#define CX_CASE(T, B, C) return launch_cross<T, B, C>(a, c->first, c->requests, (int)tiles, clusters, whole, s)
#define CX_WIDTHS(T, B) switch (dch) { case 1: CX_CASE(T, B, 1); case 2: CX_CASE(T, B, 2); case 3: CX_CASE(T, B, 3); default: CX_CASE(T, B, 4); }
    if (c->dtype == MB_F32) { if (bm == 16) CX_WIDTHS(float, 16) else CX_WIDTHS(float, 64) }
    if (c->dtype == MB_BF16) { if (bm == 16) CX_WIDTHS(bf16, 16) else CX_WIDTHS(bf16, 64) }
    return MB_ERR_BAD_DTYPE;
}
