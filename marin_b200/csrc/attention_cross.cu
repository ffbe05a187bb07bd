// Attention to an encoder's states in 32-bit arithmetic on the CUDA cores: float32 inputs, and bfloat16 ones of the layouts that the tensor-core
// kernels do not take (the formula and the layout of rows: cross_common.cuh).
// A block takes 32 rows (4, 8 or 16 where no request has more) (token, head of the group) of one request and kv head and walks its keys in tiles of 64 with a running maximum and sum:
//   S [rows x 64] = Q K^T  each thread 4 rows x 4 keys (up to 16 rows: 1 x 4), four elements of d a step from shared memory, in pairs;
//   P = exp2(S - m)        rows over 16 lanes; P through shared memory;
//   O [rows x d] += P V    each thread its rows x d / 16 columns, in registers, in pairs; four keys a step.
// A tile's values are asked for (cp.async) before S, the next tile's keys before the softmax, the places of their rows a tile earlier.
// Work split: the source is cut into up to eight chunks by its own length alone, a cluster's blocks take one each and add their partial results in
// shared memory in chunk order.  A row's arithmetic depends on its request's source and its range only, not on the batch, the portion or the tile: the same bits.
// Bound by shared memory and by latency: for 16 multiply-add pairs twice, a thread asks for eight times 16 bytes, a warp's 512 bytes come at 128 a cycle, so the four warps of an SM
// wait twice as long for them as their multiply-adds take; the rest are a tile's four barriers at 2 to 4 blocks an SM.  Five requests of 370 tokens in all, 16 heads of 64 over
// 2,908 positions 74 us (105 with tiles of 64 rows, page lookups in the loads and idle blocks that wait for their cluster; 82 with the weights read one by one, in pairs,
// instead of four at a time); four of 300 tokens, 32 heads of 128 over 600 positions 480 us, 25 TFLOP/s, where the scores' products take 155, the values' 100 and the copies 100
// that the others do not cover.  Larger shares a thread (8 x 4, 8 x 8 sums) want registers that leave too few warps: 64 rows of 128 threads 78 and 567, of 256 threads 76 and 520,
// of 64 threads 155 and 1,317; 32 rows of 64 threads 84 and 654; 2 x 8 sums (eight lanes a row) 90 and 568.  Rows copied whole by one thread each (cp.async.bulk) with two
// barriers a tile instead of four 74 and 465, and 116 for 110 with one request of 300 tokens.
// bfloat16 comes element by element through registers, not by cp.async: four of 300 tokens, 32 heads of 128 over 600 positions (pages of 8) 692 us, 480 in float32.
#define MB_LIB "attention_cross"
#define MB_LIB_ID 42
#include "cross_common.cuh"
#include "mma_helpers.cuh"
#include "pair_math.cuh"

#define CX_BN 64
#define CX_CHUNK 512               // keys a chunk at least: below that a block's tiles cost less than the cluster's meeting
#define CX_CHUNKS 8
#define CX_PSTRIDE (CX_BN + 4)

__host__ __device__ __forceinline__ int cross_chunks(int len) {
    int c = 1;
    while (c < CX_CHUNKS && c * CX_CHUNK < len) c <<= 1;
    return c;
}

// Four elements of a row of d, from element c on, as float32 into shared memory; zeros where there is no row and past d.
template <typename T>
__device__ __forceinline__ void cross_four(float* to, const T* row, int c, int d, bool whole) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (row != nullptr && c < d) {
        if (sizeof(T) == 4 && whole) { cp_async16(to, row + c); return; }
        v.x = to_f32(row[c]);
        if (c + 1 < d) v.y = to_f32(row[c + 1]);
        if (c + 2 < d) v.z = to_f32(row[c + 2]);
        if (c + 3 < d) v.w = to_f32(row[c + 3]);
    }
    *reinterpret_cast<float4*>(to) = v;
}
// 64 keys' (or values') rows of one kv head, rows LD apart, from the elements that `places` names (-1: zeros).
template <typename T, int LD, int THREADS>
__device__ __forceinline__ void cross_tile(float* dst, const CrossArgs& a, const void* cache, const long long* places, bool whole) {
    constexpr int PIECES = (LD - 4) / 4;
#pragma unroll 4
    for (int i = threadIdx.x; i < CX_BN * PIECES; i += THREADS) {
        const int row = i / PIECES, c = (i % PIECES) * 4;
        const long long place = places[row];
        cross_four<T>(dst + row * LD + c, place >= 0 ? (const T*)cache + place : nullptr, c, a.d, whole);
    }
    cp_async_commit();
}

// Registers: four blocks of 256 threads an SM where shared memory has room for them (16 rows, heads up to 64; the rows worked out again would otherwise ask for more than the loop
// does), and as many as there are for heads over 192, where it has room for one block (100 tokens of 8 heads of 256 over 500 positions, three requests: 108 us, 116 with 168).
template <typename T, int BM, int THREADS, int DCH>
__global__ void __launch_bounds__(THREADS, THREADS == 256 && DCH == 1 ? 4 : DCH == 4 ? 1 : 0) attention_cross_kernel(const __grid_constant__ CrossArgs arg, int first_request, int requests, int max_tiles, int whole, int q_whole) {
    constexpr int RM = BM * 16 / THREADS, LD = DCH * 64 + 4;
    extern __shared__ __align__(16) float cx_smem[];
    float* sQ = cx_smem;                                            // [BM][LD]; later the partial results
    float* sK = sQ + BM * LD;
    float* sV = sK + CX_BN * LD;
    float* sP = sV + CX_BN * LD;                                    // [BM][CX_PSTRIDE]
    __shared__ float s_m[BM], s_l[BM];
    __shared__ int s_lo[BM], s_hi[BM], s_first, s_last;
    __shared__ long long s_place[2][CX_BN];                         // where a tile's rows begin in the caches
    PDL_ENTER();
    CrossArgs a = arg;
    a.q = pdl_fresh((const char*)a.q); a.k_cache = pdl_fresh((const char*)a.k_cache); a.v_cache = pdl_fresh((const char*)a.v_cache);
    a.block_table = pdl_fresh(a.block_table); a.lens = pdl_fresh(a.lens); a.cu_tokens = pdl_fresh(a.cu_tokens); a.spans = pdl_fresh(a.spans);
    const int2 which = cross_tile_of(a, first_request, requests, a.G, BM, max_tiles, blockIdx.x / a.K);       // (a tile's heads side by side)
    if (which.x < 0) return;
    const int r = which.x, tile = which.y, kh = blockIdx.x % a.K;
    const int rank = blockIdx.z, t0 = a.cu_tokens[r], rows = (a.cu_tokens[r + 1] - t0) * a.G, row0 = tile * BM;
    if (row0 >= rows) return;                                       // (all blocks of a cluster)
    const int len = max(0, min(a.lens[r], a.max_pages << a.page_shift));
    const int chunks = min(cross_chunks(len), (int)gridDim.z), H = a.K * a.G;
    if (rank >= chunks) return;                                     // (a cluster's barriers wait for those that are there)
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
    for (int i = tid; i < BM * (LD / 4 - 1); i += THREADS) {
        const int row = i / (LD / 4 - 1), c = (i % (LD / 4 - 1)) * 4, at = row0 + row;
        cross_four<T>(sQ + row * LD + c, at < rows ? (const T*)a.q + (size_t)(t0 + at / a.G) * a.q_stride + (size_t)(kh * a.G + at % a.G) * a.d : nullptr, c, a.d, q_whole);
    }
    cp_async_commit();
    __syncthreads();
    const int tiles = (len + CX_BN - 1) / CX_BN, per = (tiles + chunks - 1) / chunks;
    const int from = max(rank * per, s_first / CX_BN);
    const int to = s_last > s_first ? min(min(tiles, (rank + 1) * per), (s_last + CX_BN - 1) / CX_BN) : 0;
    const float sl2 = a.scale * 1.4426950408889634f;
    float m[RM], l[RM];
    uint64_t o[RM][DCH][2];                                         // four columns as two pairs
    int lo[RM], hi[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        m[i] = -INFINITY; l[i] = 0.0f;
        lo[i] = s_lo[ty * RM + i]; hi[i] = s_hi[ty * RM + i];
#pragma unroll
        for (int c = 0; c < DCH; ++c) o[i][c][0] = o[i][c][1] = 0;
    }
    const int first = s_first, last = s_last, steps = (a.d + 3) / 4;
    // Where the rows of a tile lie is looked up two tiles ahead of its keys (a page's number is a round trip to memory), a thread a row.
    auto page_of = [&](int kt) {
        const int key = kt * CX_BN + tid;
        return tid < CX_BN && kt < to && key >= first && key < last ? table[key >> a.page_shift] : -1;
    };
    auto place_rows = [&](int kt, int page) {
        const int key = kt * CX_BN + tid;
        if (tid < CX_BN) s_place[kt & 1][tid] = page < 0 ? -1 : ((((long long)page * a.K + kh) << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * a.d;
    };
    if (from < to) {
        place_rows(from, page_of(from));
        __syncthreads();
        cross_tile<T, LD, THREADS>(sK, a, a.k_cache, s_place[from & 1], whole);
    }
    int page = page_of(from + 1);
    for (int kt = from; kt < to; ++kt) {
        const int key0 = kt * CX_BN;
        cross_tile<T, LD, THREADS>(sV, a, a.v_cache, s_place[kt & 1], whole);
        place_rows(kt + 1, page);
        page = page_of(kt + 2);
        cp_async_wait<1>();
        __syncthreads();
        // (elements of d in pairs: even ones' sum and odd ones')
        uint64_t s2[RM][4];
#pragma unroll
        for (int i = 0; i < RM; ++i) s2[i][0] = s2[i][1] = s2[i][2] = s2[i][3] = 0;
#pragma unroll 4
        for (int x = 0; x < steps; ++x) {
            ulonglong2 kv[4], qv[RM];
#pragma unroll
            for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const ulonglong2*>(sK + (tx + 16 * j) * LD + 4 * x);
#pragma unroll
            for (int i = 0; i < RM; ++i) qv[i] = *reinterpret_cast<const ulonglong2*>(sQ + (ty * RM + i) * LD + 4 * x);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s2[i][j] = fma_pair(qv[i].x, kv[j].x, s2[i][j]);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s2[i][j] = fma_pair(qv[i].y, kv[j].y, s2[i][j]);
        }
        float s[RM][4];
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float even, odd;
                of_pair(s2[i][j], even, odd);
                s[i][j] = even + odd;
            }
        __syncthreads();
        if (kt + 1 < to) cross_tile<T, LD, THREADS>(sK, a, a.k_cache, s_place[(kt + 1) & 1], whole);
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
            const uint64_t corrs = pair_of(corr, corr);
#pragma unroll
            for (int c = 0; c < DCH; ++c) { o[i][c][0] = mul_pair(o[i][c][0], corrs); o[i][c][1] = mul_pair(o[i][c][1], corrs); }
        }
        cp_async_wait<1>();
        __syncthreads();
#pragma unroll 4
        for (int j = 0; j < CX_BN; j += 4) {
            float4 pv[RM];
#pragma unroll
            for (int i = 0; i < RM; ++i) pv[i] = *reinterpret_cast<const float4*>(sP + (ty * RM + i) * CX_PSTRIDE + j);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                uint64_t w[RM];
#pragma unroll
                for (int i = 0; i < RM; ++i) { const float p = jj == 0 ? pv[i].x : jj == 1 ? pv[i].y : jj == 2 ? pv[i].z : pv[i].w; w[i] = pair_of(p, p); }
#pragma unroll
                for (int c = 0; c < DCH; ++c) {
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sV + (j + jj) * LD + c * 64 + tx * 4);
#pragma unroll
                    for (int i = 0; i < RM; ++i) {
                        o[i][c][0] = fma_pair(w[i], v.x, o[i][c][0]);
                        o[i][c][1] = fma_pair(w[i], v.y, o[i][c][1]);
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
        for (int c = 0; c < DCH; ++c) *reinterpret_cast<ulonglong2*>(sQ + row * LD + c * 64 + tx * 4) = make_ulonglong2(o[i][c][0], o[i][c][1]);
    }
    if (gridDim.z > 1) cross_cluster_sync(); else __syncthreads();
    // block `rank` finishes rows rank, rank + chunks, ...: a warp a row, the chunks in their order
    constexpr int PIECES = DCH > 2 ? 2 : 1, AT_ONCE = BM == 32 ? 4 : 2;
    const int warp = tid >> 5, lane = tid & 31;
    bool looked = false;
    int2 odd_values = make_int2(0, 0);
    for (int row = rank + warp * chunks; row < BM; row += THREADS / 32 * chunks) {
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
        if (a.spans != nullptr && __any_sync(0xffffffffu, odd) && cross_sum_speaks(sum)) {
            const int2 range = make_int2(s_lo[row], s_hi[row]);
            if (cross_whole<T>(arg)) {
                if (!looked) odd_values = cross_odd_values<T, PIECES, true>(arg, kh, r, first, last);
                if (cross_not_its_own(odd_values, range)) { __syncwarp(); cross_row_alone<T, PIECES, AT_ONCE, true>(arg, t, head, r, range); }
            } else {
                if (!looked) odd_values = cross_odd_values<T, PIECES, false>(arg, kh, r, first, last);
                if (cross_not_its_own(odd_values, range)) { __syncwarp(); cross_row_alone<T, PIECES, 1, false>(arg, t, head, r, range); }
            }
            looked = true;
        }
    }
    if (gridDim.z > 1) cross_cluster_sync();                        // (a block's shared memory is read until here)
}

template <typename T, int BM, int THREADS, int DCH>
static int launch_cross(const CrossArgs& a, int first_request, int requests, CrossGrid grid, int clusters, int whole, int q_whole, cudaStream_t s) {
    constexpr int LD = DCH * 64 + 4;
    const size_t smem = ((size_t)(BM + 2 * CX_BN) * LD + BM * CX_PSTRIDE) * sizeof(float);
    static LaunchSmem allowed;
    const int rc = allowed.allow(attention_cross_kernel<T, BM, THREADS, DCH>, smem);
    if (rc != 0) return rc;
    return launch_kernel(attention_cross_kernel<T, BM, THREADS, DCH>, dim3((unsigned)grid.blocks * a.K, 1, clusters), dim3(THREADS), smem, s, clusters, a, first_request,
                         requests, grid.max_tiles, whole, q_whole);
}

MB_API int mb_attention_cross(const CrossCall* c, cudaStream_t s) {
    if (c->requests <= 0 || c->max_query <= 0) return 0;
    if (!cross_call_fits(c) || c->d > 256) return MB_ERR_BAD_SIZE;
    const CrossArgs a = cross_args(c);
    const int whole = c->dtype == MB_F32 && a.d % 4 == 0 && (((uintptr_t)c->k_cache | (uintptr_t)c->v_cache) & 15) == 0;
    const int q_whole = c->dtype == MB_F32 && a.d % 4 == 0 && ((uintptr_t)c->q & 15) == 0 && c->q_stride % 4 == 0;
    // Few rows a request (single tokens): tiles of as few, for every row that is not there asks shared memory for keys and values all the same.  (Float32, tiles of 4 rows
    // against tiles of 16: 8 single tokens over 2,000 positions, 16 heads of 64 49 and 92 us; 32 over 100 to 2,000 113 and 233; 32 over 600 positions,
    // 32 heads of 128 over 8 81 and 117; 8 over 577 positions of the latter 40 and 39.)
    const long long rows = (long long)c->max_query * a.G;
    const int bm = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    const CrossGrid grid = cross_grid(c, a.G, bm);
    if (grid.blocks * a.K > 0x7fffffffLL) return MB_ERR_BAD_SIZE;
    const int clusters = cross_chunks(c->longest), dch = (a.d + 63) / 64;
#define CX_CASE(T, B, N, C) return launch_cross<T, B, N, C>(a, c->first, c->requests, grid, clusters, whole, q_whole, s)
#define CX_WIDTHS(T, B, N) switch (dch) { case 1: CX_CASE(T, B, N, 1); case 2: CX_CASE(T, B, N, 2); case 3: CX_CASE(T, B, N, 3); default: CX_CASE(T, B, N, 4); }
#define CX_ROWS(T) { if (bm == 4) CX_WIDTHS(T, 4, 64) if (bm == 8) CX_WIDTHS(T, 8, 128) if (bm == 16) CX_WIDTHS(T, 16, 256) CX_WIDTHS(T, 32, 128) }
    if (c->dtype == MB_F32) CX_ROWS(float)
    if (c->dtype == MB_BF16) CX_ROWS(bf16)
    return MB_ERR_BAD_DTYPE;
}
