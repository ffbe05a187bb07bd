// Attention of single tokens to an encoder's states, bfloat16, up to eight query heads a kv head, pages of at least 16 positions (the formula:
// cross_common.cuh).  Compiled per head size (-DHEAD_DIM, a multiple of 16 up to 128).
//
// Every key and value of a request is read once for all heads of its kv head, so the bytes bound it.  A cluster of up to eight blocks takes one request and kv
// head, each block an equal run of the positions (requests of a batch have sources of all lengths: shares by length keep the blocks of a cluster equal, where runs
// of a fixed length leave most blocks of short ones idle); its four warps take stages of 16 positions in turn, each through a ring of its own (cp.async into padded
// rows, two stages on their way a warp), no barrier of the block in the loop.  The query heads are rows 0..7 of mma.sync.m16n8k16:
//   S = Q K^T   rows 8..15 of Q are zeros;
//   O = P V     rows 0..7 hold a weight rounded to bfloat16, rows 8..15 what the rounding took off, rounded in turn: O's rows r and r + 8 add up to the weights'
//               product at 16 bits of a weight, for no more products.  (Where a value is infinite the first alone count: what is left of a weight may be 0.)
// Maximum, sum and O are float32; warps, then blocks (in shared memory, rank order), add up theirs scaled to the common maximum.
// Positions outside the row's range are zeros in shared memory (asked for with no bytes), so what lies there does not matter.
// Measured on B200: 64 requests of 500 to 4,100 positions, 8 kv heads of 128 (547 MB) 91 us, 6.0 TB/s, 91 % of the copy rate; one request of 577 positions 6 us in a graph, its chain of
// dependent loads (lengths, pages, keys), products and the cluster's meeting.
#define MB_LIB "attention_cross_decode"
#define MB_LIB_ID 44
#include "cross_common.cuh"
#include "mma_helpers.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<multiple of 16, at most 128>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 128, "heads in steps of 16 up to 128");

#define D HEAD_DIM
#ifndef XD_WARPS
#define XD_WARPS 4
#endif
#define XD_KEYS 16                               // positions of a stage
#ifndef XD_STAGES
#define XD_STAGES 2
#endif
#define XD_LD (D + 8)                            // elements of a padded row: ldmatrix without bank conflicts
#define XD_STAGE_BYTES (2 * XD_KEYS * XD_LD * 2)
#define XD_RING (XD_STAGES * XD_STAGE_BYTES)
#define XD_SMEM (XD_WARPS * XD_RING)
// More blocks than fit at once (three an SM), each a request's: the longest sources first, or the launch ends with a few of them (B200, 64 requests of 500 to 4,100 positions, 8 kv
// heads of 128: 89 us, 103 in the order of requests; where all have 577 the search for the order costs 32 us against 31).
#define XD_AT_ONCE (3 * 148)
#define XD_SORTED 128                            // requests at most that a block looks through for its own
static_assert(8 * D * 4 <= XD_RING, "a warp's O is written over its ring");

__device__ __forceinline__ float xd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16_or_zeros(void* dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}

__global__ void __launch_bounds__(XD_WARPS * 32) attention_cross_decode_kernel(CrossArgs a, int first_request, int sorted) {
    extern __shared__ __align__(16) uint8_t xd_smem[];
    __shared__ float w_m[XD_WARPS][8], w_l[XD_WARPS][8], c_m[8], c_l[8];
    __shared__ __align__(16) float c_o[8 * D];
    __shared__ __align__(16) int s_len[XD_SORTED];
    __shared__ int4 s_mine;
    PDL_ENTER();
    a.q = pdl_fresh((const char*)a.q); a.k_cache = pdl_fresh((const char*)a.k_cache); a.v_cache = pdl_fresh((const char*)a.v_cache);
    a.block_table = pdl_fresh(a.block_table); a.lens = pdl_fresh(a.lens); a.cu_tokens = pdl_fresh(a.cu_tokens); a.spans = pdl_fresh(a.spans);
    const int kh = sorted > 0 ? blockIdx.x % a.K : blockIdx.y, rank = blockIdx.z, cluster = gridDim.z, G = a.G, tid = threadIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int r = first_request + blockIdx.x, t, tokens, len;
    if (sorted > 0) {
        // the requests by length, the longest first, a request's heads side by side: every thread counts the requests that come ahead of its own
        static_assert(XD_SORTED == XD_WARPS * 32, "a thread a request");
        const int at = first_request + min(tid, sorted - 1), mine = tid < sorted ? max(0, a.lens[at]) : -1, begins = a.cu_tokens[at], ends = a.cu_tokens[at + 1];
        s_len[tid] = mine;
        __syncthreads();
        int ahead = 0;
#pragma unroll 4
        for (int i = 0; i < sorted; i += 4) {
            const int4 v = *reinterpret_cast<const int4*>(s_len + i);
            const int other[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) ahead += other[e] > mine || (other[e] == mine && i + e < tid);
        }
        if (tid < sorted && ahead == (int)(blockIdx.x / a.K)) s_mine = make_int4(tid, begins, ends - begins, mine);
        __syncthreads();
        r = first_request + s_mine.x; t = s_mine.y; tokens = s_mine.z; len = s_mine.w;
    } else {
        t = a.cu_tokens[r]; tokens = a.cu_tokens[r + 1] - t; len = a.lens[r];
    }
    len = max(0, min(len, a.max_pages << a.page_shift));
    if (tokens <= 0) return;                                        // (a padded request: all blocks of its clusters)
    const int2 range = cross_range(a, t, len);
    const int* table = a.block_table + (size_t)r * a.max_pages;
    // stages of 16 positions: the block's share, and of it every fourth for this warp
    const int stage0 = range.x / XD_KEYS, stages = range.y > range.x ? (range.y + XD_KEYS - 1) / XD_KEYS - stage0 : 0;
    const int share = (stages + cluster - 1) / cluster, mine0 = stage0 + rank * share, mine_n = max(0, min(share, stages - rank * share));
    const int steps = mine_n > warp ? (mine_n - warp + XD_WARPS - 1) / XD_WARPS : 0;

    uint8_t* ring = xd_smem + (size_t)warp * XD_RING;
    const size_t head_rows = (size_t)kh << a.page_shift, page_rows = (size_t)a.K << a.page_shift;
    // page of step i, for the 32 steps around: a lane a step
    int pages = 0;
    auto look_up = [&](int i) {
        const int step = i + lane;
        pages = step < steps ? table[((mine0 + warp + step * XD_WARPS) * XD_KEYS) >> a.page_shift] : 0;
    };
    auto issue = [&](int i) {
        if (i < steps) {
            if ((i & 31) == 0) look_up(i);
            const int key0 = (mine0 + warp + i * XD_WARPS) * XD_KEYS;
            const size_t row0 = (size_t)__shfl_sync(0xffffffffu, pages, i & 31) * page_rows + head_rows + (size_t)(key0 & ((1 << a.page_shift) - 1));
            const bf16 *ks = (const bf16*)a.k_cache + row0 * D, *vs = (const bf16*)a.v_cache + row0 * D;
            bf16* dst = reinterpret_cast<bf16*>(ring + (size_t)(i % XD_STAGES) * XD_STAGE_BYTES);
            constexpr int PIECES = D / 8;
#pragma unroll
            for (int x = lane; x < XD_KEYS * PIECES; x += 32) {
                const int row = x / PIECES, piece = x % PIECES;
                const bool there = key0 + row >= range.x && key0 + row < range.y;
                cp_async16_or_zeros(dst + row * XD_LD + piece * 8, ks + row * D + piece * 8, there);
                cp_async16_or_zeros(dst + (XD_KEYS + row) * XD_LD + piece * 8, vs + row * D + piece * 8, there);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < XD_STAGES; ++i) issue(i);

    // the query rows straight into the MMA's A fragments: lane l holds row l / 4, columns 2 (l % 4) + {0, 1} and + 8 of every 16
    uint32_t qa[D / 16][4];
    {
        const int row = lane >> 2;
        const bf16* q = (const bf16*)a.q + (size_t)t * a.q_stride + (size_t)(kh * G + (row < G ? row : 0)) * D + 2 * (lane & 3);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            qa[kk][0] = row < G ? *reinterpret_cast<const uint32_t*>(q + kk * 16) : 0u;
            qa[kk][2] = row < G ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8) : 0u;
            qa[kk][1] = qa[kk][3] = 0u;
        }
    }
    const float sl2 = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;                                  // of this lane's row (query head lane / 4)
    float o[D / 8][4];                                              // [0], [1]: row lane / 4; [2], [3]: what the rounded weights left
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    for (int i = 0; i < steps; ++i) {
        cp_async_wait<XD_STAGES - 1>();
        __syncwarp();
        const int key0 = (mine0 + warp + i * XD_WARPS) * XD_KEYS;
        const bf16* sK = reinterpret_cast<const bf16*>(ring + (size_t)(i % XD_STAGES) * XD_STAGE_BYTES);
        const bf16* sV = sK + XD_KEYS * XD_LD;
        float sc[2][4];
        sc[0][0] = sc[0][1] = sc[0][2] = sc[0][3] = sc[1][0] = sc[1][1] = sc[1][2] = sc[1][3] = 0.0f;
        const uint32_t k_addr = (uint32_t)__cvta_generic_to_shared(sK + ((lane & 7) + (lane >> 4) * 8) * XD_LD + ((lane >> 3) & 1) * 8);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4(k_addr + kk * 32, b0, b1, b2, b3);
            mma_bf16_16816(sc[0], qa[kk], b0, b1);
            mma_bf16_16816(sc[1], qa[kk], b2, b3);
        }
        float s[4] = {sc[0][0] * sl2, sc[0][1] * sl2, sc[1][0] * sl2, sc[1][1] * sl2};
        if (key0 < range.x || key0 + XD_KEYS > range.y) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = key0 + 2 * (lane & 3) + (j >> 1) * 8 + (j & 1);
                if (key < range.x || key >= range.y) s[j] = -INFINITY;
            }
        }
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (__any_sync(0xffffffffu, mx > m)) {                      // (seldom after the first stages)
            const float m_new = fmaxf(m, mx), corr = xd_exp2(m - (m_new == -INFINITY ? 0.0f : m_new));
            m = m_new;
            l *= corr;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) { o[c][0] *= corr; o[c][1] *= corr; o[c][2] *= corr; o[c][3] *= corr; }
        }
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < 4; ++j) { s[j] = xd_exp2(s[j] - base); l += s[j]; }
        uint32_t pa[4];
        pa[0] = pack_bf16(s[0], s[1]);
        pa[2] = pack_bf16(s[2], s[3]);
        const float2 h0 = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&pa[0])), h1 = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&pa[2]));
        pa[1] = pack_bf16(s[0] - h0.x, s[1] - h0.y);
        pa[3] = pack_bf16(s[2] - h1.x, s[3] - h1.y);
        const uint32_t v_addr = (uint32_t)__cvta_generic_to_shared(sV + ((lane & 7) + ((lane >> 3) & 1) * 8) * XD_LD + (lane >> 4) * 8);
#pragma unroll
        for (int c = 0; c < D / 8; c += 2) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4_trans(v_addr + c * 16, b0, b1, b2, b3);
            mma_bf16_16816(o[c], pa, b0, b1);
            mma_bf16_16816(o[c + 1], pa, b2, b3);
        }
        __syncwarp();                                               // the stage is free
        issue(i + XD_STAGES);
    }
    cp_async_wait<0>();
    __syncwarp();
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    {
        float* mine = reinterpret_cast<float*>(ring) + (lane >> 2) * D + 2 * (lane & 3);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)                             // (a value that is infinite is so by the rounded weights' product: what they left may be 0 or negative)
            *reinterpret_cast<float2*>(mine + c * 8) = make_float2(fabsf(o[c][0]) <= 3.0e38f ? o[c][0] + o[c][2] : o[c][0], fabsf(o[c][1]) <= 3.0e38f ? o[c][1] + o[c][3] : o[c][1]);
        if ((lane & 3) == 0) { w_m[warp][lane >> 2] = m; w_l[warp][lane >> 2] = l; }
    }
    __syncthreads();
    // the block's result, then the cluster's
    for (int x = threadIdx.x; x < G * D; x += XD_WARPS * 32) {
        const int row = x / D;
        float top = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < XD_WARPS; ++w) top = fmaxf(top, w_m[w][row]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < XD_WARPS; ++w) {
            const float f = xd_exp2(w_m[w][row] - base);
            sum = fmaf(f, w_l[w][row], sum);
            v = fmaf(f, reinterpret_cast<const float*>(xd_smem + (size_t)w * XD_RING)[x], v);
        }
        if (cluster == 1) {
            ((bf16*)a.out)[((size_t)t * a.K * G + kh * G) * D + x] = __float2bfloat16_rn(range.y > range.x ? v / sum : 0.0f);
        } else {
            c_o[x] = v;
            if (x % D == 0) { c_m[row] = top; c_l[row] = sum; }
        }
    }
    if (cluster == 1) return;
    cross_cluster_sync();
    for (int row = rank + warp * cluster; row < G; row += XD_WARPS * cluster) {             // a warp a row, four columns a lane
        float sum;
        const float factor = cross_factor<false>(&c_m[row], &c_l[row], cluster, sum);
        const float4 v = cross_join4(c_o + row * D + min(4 * lane, D - 4), factor, cluster);
        const bool sees = range.y > range.x;
        if (4 * lane < D) {
            uint2 w;
            w.x = pack_bf16(sees ? v.x / sum : 0.0f, sees ? v.y / sum : 0.0f);
            w.y = pack_bf16(sees ? v.z / sum : 0.0f, sees ? v.w / sum : 0.0f);
            reinterpret_cast<uint2*>((bf16*)a.out + ((size_t)t * a.K * G + kh * G + row) * D)[lane] = w;
        }
    }
    cross_cluster_sync();                                           // (a block's shared memory is read until here)
}

// Requests of one token each.
MB_API int mb_attention_cross_decode(const CrossCall* c, cudaStream_t s) {
    if (c->requests <= 0) return 0;
    if (!cross_call_fits(c) || c->d != D || c->dtype != MB_BF16 || c->page_size < XD_KEYS || c->H / c->K > 8 || ((uintptr_t)c->q & 3) != 0 || ((uintptr_t)c->out & 7) != 0 || c->q_stride % 2 != 0 ||
        (((uintptr_t)c->k_cache | (uintptr_t)c->v_cache) & 15) != 0 || !chunks_fit(c->chunks))
        return MB_ERR_BAD_SIZE;
    static LaunchSmem allowed;
    const int rc = allowed.allow(attention_cross_decode_kernel, XD_SMEM);
    if (rc != 0) return rc;
    const long long pairs = (long long)c->requests * c->K;
    if (pairs > 0x7fffffffLL) return MB_ERR_BAD_SIZE;
    const int sorted = c->requests > 1 && c->requests <= XD_SORTED && c->chunks == 1 && pairs > XD_AT_ONCE ? c->requests : 0;
    return launch_kernel(attention_cross_decode_kernel, sorted > 0 ? dim3((unsigned)pairs, 1, c->chunks) : dim3(c->requests, c->K, c->chunks), dim3(XD_WARPS * 32), XD_SMEM, s, c->chunks, cross_args(c), c->first, sorted);
}
