// Attention to an encoder's states on the 5th-generation tensor cores (tcgen05 / TMEM), bfloat16, portions of any length; the formula and the layout
// of rows are in cross_common.cuh.  Compiled per head size (-DHEAD_DIM, a multiple of 16 up to 128); any number of query heads a kv head up to 128.
//
// No mask depends on the order of tokens, so a tile's 128 rows are (token, query head of the group) pairs: 128 / G tokens of all heads that share a kv
// head, one TMA box of [tokens][G][64 columns]; a portion of seven tokens fills as much of a tile as it can, and keys are fetched once for all of them.
// A block works on one tile at a time, in blocks of 64 keys:
//   S = Q K^T     tcgen05.mma 128 x 64 x d, operands in shared memory (TMA, 128-byte swizzle, K-major), S in one of two buffers in tensor memory;
//   P = 2^(S - m) a thread a row: 64 scores by tcgen05.ld, maximum, exponentials in pairs, P as bfloat16 over the row's own scores (tcgen05.st).  The
//                 maximum that O and the sum are scaled by follows the true one only when that has moved by more than 8 (2^8, harmless in float32);
//   O += P V      tcgen05.mma with P from tensor memory, V as it lies in the cache ([key][d], an MN-major operand), O in d columns.
// With two buffers of scores the rows work on one while the other's P V and next S are made.  Two blocks an SM (256 columns of tensor memory and about 100 KB each):
// one's barriers, first loads and last stores are time in which the other works.
// Warps 0..3 are the rows, 4 loads Q and K, 5 loads V, 6 issues the products.  Sums, maxima and O are float32; P is rounded to
// bfloat16 as the products' operand (its error, at most 2^-8 of a weight, is that of the rounding of the result; the sum takes the weights before it).
// Measured on B200 (heads of 128, four prompts of 1,024 tokens of 32 heads over 4,096 positions, 275 GFLOP): 235 us (277 over
// seconds, at the power limit's clock of 1.6 GHz).  What was tried: two tiles a block over the same
// keys, one block an SM, with blocks of 128 keys (267 us) or 64 (262), with two threads a row (258 to 272), an issuer for both (274): slower, although a
// key then comes for twice as many rows; blocks that stay and take tile after tile, loads ahead into the next (265); the special-function unit's exponentials by a
// polynomial for a part of the scores (no gain).
//
// Few rows: the blocks of keys are cut over a cluster of up to eight blocks, which add their partial O in shared memory in rank order.
// What is not there: keys past the source are masked; values past it are zeros (0 * NaN is NaN): whole boxes by copies outside the tensor, the box that
// the source ends in by plain stores.  Waits are bounded and record a code in *error_flag.
#define MB_LIB "attention_cross_tc"
#define MB_LIB_ID 43
#include "tc_common.cuh"
#include "cross_common.cuh"
#include "pair_math.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<multiple of 16, at most 128>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 128, "heads in steps of 16 up to 128");

#define D HEAD_DIM
#define NH ((D + 63) / 64)                       // 64-column panels of a row (copies zero-fill past the row's end)
#define XT_BM 128
#define XT_BN 64                                 // keys of a block
#define XT_TILE (NH * XT_BM * 128)               // bytes of a tile of queries
#define XT_KV (NH * XT_BN * 128)                 // bytes of a block of keys, or of values
#define XT_OLD (D + 4)                           // floats between rows of O for the cluster
#define XT_BARS 512
// 16-byte piece c of row r of a tile's results in shared memory: rows of whole 128 bytes swizzled, others a piece apart, so that neither a thread's row nor a
// row across threads meets a bank twice
#if HEAD_DIM % 64 == 0
#define XT_STAGED(r, c) ((r) * (D / 8) + ((c) ^ ((r) & 7)))
#else
#define XT_STAGED(r, c) ((r) * (D / 8 + 1) + (c))
#endif
static_assert(D % 64 == 0 || XT_BM * (D * 2 + 16) <= XT_TILE, "a tile's results fit its queries' memory");
#define XT_STAGES (NH == 1 ? 4 : 2)              // blocks of keys, and of values, on their way
#define XT_SMEM (XT_TILE + 2 * XT_STAGES * XT_KV + XT_BARS)
#define XT_TMEM 256                              // two buffers of scores (64 columns each), then O
#define XT_O_COL 128
#define XT_THREADS 256                           // warps 0..3 the rows, 4 loads Q and K, 5 V, 6 issues the products
static_assert(XT_BM * XT_OLD * 4 <= XT_TILE + 2 * XT_STAGES * XT_KV, "partial results fit the tile's memory");
static_assert(2 * (XT_SMEM + 1024 + XT_BM * 20 + 512) <= 233472, "two blocks an SM");
#define XT_MAX_CLUSTER 8
#define XT_SMS 148
struct CrossTc {
    CrossArgs a;
    int* error_flag;
    int first_request, requests, max_tiles, cache_rows;
};

__device__ __forceinline__ float xt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 32 columns of this thread's lane; nothing of v may be used before tmem_ld_wait.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
// (the values go through it: the compiler must not use a register of the load ahead of the wait)
__device__ __forceinline__ void tmem_ld_wait(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                   "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                   "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16_bits(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
          "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
          "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}

__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for a phase; gives up at once if another thread of the block already gave up (`*abort`), and says so itself when its own time limit passes.
// (The clock is asked only where the phase was not there at once: reading it cost as much as the wait.)
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort, int* error_flag, int code) {
    if (mbar_try(bar, parity)) return true;
    const long long start = clock64();
    for (unsigned polls = 1;; ++polls) {
        if (mbar_try(bar, parity)) return true;
        if ((polls & 31) == 0) {
            if (*abort) return false;
            if (clock64() - start > TC_WAIT_LIMIT) { *abort = 1; atomicExch(error_flag, code); return false; }
        }
    }
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* error_flag, int code) {
    return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort, error_flag, code));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
// The MMA with its A operand in tensor memory (row m in lane m, two bf16 per 32-bit column) and B in shared memory.
__device__ __forceinline__ void umma_bf16_tmem_a(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t elected) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}

__global__ void __launch_bounds__(XT_THREADS, 2) attention_cross_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CrossTc arg) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;                                             // [panel][128 rows][128 B]
    uint8_t* sK = sQ + XT_TILE;                                     // [stage][panel][64 rows][128 B]
    uint8_t* sV = sK + XT_STAGES * XT_KV;
    uint64_t* bars = (uint64_t*)(sV + XT_STAGES * XT_KV);
    uint64_t* q_full = bars;
    uint64_t* s_full = bars + 1;                                    // [buffer] scores are there
    uint64_t* p_full = bars + 3;                                    // [buffer] weights are there (four warps arrive)
    uint64_t* o_done = bars + 5;                                    // [block % 4] P V of the block's weights is done
    uint64_t* drained = bars + 9;
    uint64_t* k_full = bars + 10;                                   // [stage]
    uint64_t* k_free = k_full + XT_STAGES;
    uint64_t* v_full = k_free + XT_STAGES;
    uint64_t* v_free = v_full + XT_STAGES;
    uint32_t* tmem_slot = (uint32_t*)(v_free + XT_STAGES);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    __shared__ float s_m[XT_BM], s_l[XT_BM];
    __shared__ int2 s_range[XT_BM];
    __shared__ int s_to[XT_BM];                                     // where a row's result begins, from the block's first token on; -1: no row
    __shared__ int s_seen[2][4];                                    // [first, end) that each warp's rows see
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    PDL_ENTER_EARLY();
    CrossArgs a = arg.a;
    a.q = pdl_fresh((const char*)a.q); a.v_cache = pdl_fresh((const char*)a.v_cache); a.k_cache = pdl_fresh((const char*)a.k_cache);
    a.block_table = pdl_fresh(a.block_table); a.lens = pdl_fresh(a.lens); a.cu_tokens = pdl_fresh(a.cu_tokens); a.spans = pdl_fresh(a.spans);
    int* error_flag = arg.error_flag;
    const int rank = blockIdx.z, cluster = gridDim.z, kh = blockIdx.x % a.K, G = a.G, per_tile = XT_BM / G;
    const int2 which = cross_tile_of(a, arg.first_request, arg.requests, 1, per_tile, arg.max_tiles, blockIdx.x / a.K);    // (a tile's heads side by side)
    if (which.x < 0) return;                                        // (all blocks of a cluster)
    const int r = which.x, number = which.y;
    const int tok0 = a.cu_tokens[r] + number * per_tile, left = a.cu_tokens[r + 1] - tok0;
    const int source = a.lens[r];
    if (left <= 0) return;                                          // (all blocks of a cluster)
    if ((smem_u32(smem) & 1023u) != 0) { if (tid == 0) atomicExch(error_flag, 40); return; }
    const int len = max(0, min(source, a.max_pages << a.page_shift));
    const int* table = a.block_table + (size_t)r * a.max_pages;
    if (warp == 4) {                                                // (the queries are asked for at once; the keys' range is not known yet)
        if (lane == 0) {
            mbar_init(q_full, 1); mbar_init(drained, 1);
            for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); }
            for (int i = 0; i < 4; ++i) mbar_init(&o_done[i], 1);
            for (int i = 0; i < XT_STAGES; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_free[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_free[i], 1); }
            *abort = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            mbar_expect_tx(q_full, (uint32_t)(NH * per_tile * G * 128));
            for (int p = 0; p < NH; ++p) tma_load_3d(sQ + p * (XT_BM * 128), &map_q, p * 64, kh * G, tok0, q_full);
        }
        __syncwarp();
    }
    if (warp == 7) { __syncwarp(); tmem_alloc<false>(tmem_slot, XT_TMEM); }
    // this thread's row (the first threads): tile, token, head
    const int my_tok = tid / G, my_head = kh * G + tid % G;
    const bool mine = tid < per_tile * G && my_tok < left;
    int2 range = make_int2(0, 0);
    if (mine) range = cross_range(a, tok0 + my_tok, len);
    if (warp < 4) {
        s_range[tid] = range;
        s_to[tid] = mine ? (my_tok * a.K * G + my_head) * D : -1;
        const int lowest = __reduce_min_sync(0xffffffffu, range.y > range.x ? range.x : len), highest = __reduce_max_sync(0xffffffffu, range.y);
        if (lane == 0) { s_seen[0][warp] = lowest; s_seen[1][warp] = highest; }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    int first_seen = s_seen[0][0], end_seen = s_seen[1][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) { first_seen = min(first_seen, s_seen[0][w]); end_seen = max(end_seen, s_seen[1][w]); }
    const int first_block = first_seen / XT_BN, blocks_all = end_seen > first_seen ? (end_seen + XT_BN - 1) / XT_BN - first_block : 0;
    bf16* const out0 = (bf16*)a.out + (size_t)tok0 * a.K * G * D;
    if (blocks_all == 0) {                                          // nobody here sees anything: zeros (all blocks of a cluster come here)
        if (warp == 7) { __syncwarp(); tmem_free<false>(tmem_base, XT_TMEM); }
        mbar_wait(q_full, 0);                                       // (what was asked for has to land)
        for (int x = rank * XT_THREADS + tid; x < XT_BM * (D / 8); x += cluster * XT_THREADS) {
            const int to = s_to[x / (D / 8)];
            if (to >= 0) reinterpret_cast<uint4*>(out0 + to)[x % (D / 8)] = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const int share = (blocks_all + cluster - 1) / cluster;
    const int block0 = first_block + rank * share, nblk = max(0, min(share, blocks_all - rank * share));

    const int role = warp_same(warp);                               // (the branches are then the same in all lanes for the compiler too: see elect_one)
    if (role >= 4) {
        if (role == 4 || role == 5) {
            // ---- the loaders: a lane a box (a page's rows of one panel), as soon as the block's buffer is free; where the boxes lie is looked up a block ahead ----
            const bool keys = role == 4;
            const CUtensorMap* map = keys ? &map_k : &map_v;
            uint64_t* full = keys ? k_full : v_full;
            uint64_t* freed = keys ? k_free : v_free;
            const int page = 1 << a.page_shift, rows = min(page, XT_BN), boxes = XT_BN / rows, box = lane % boxes, panel = lane / boxes;
            const bool loads = panel < NH;
            // pages of 32 boxes, a lane a box, and of the 32 after them: looked up while the ones at hand are used
            auto ids_at = [&](int x0) -> int {
                const int x = x0 + lane, key = block0 * XT_BN + x * rows;
                return x < nblk * boxes && key < len ? table[key >> a.page_shift] : -1;
            };
            int ids_from = 0, ids = ids_at(0), ids_next = ids_at(32);
            __syncwarp();
            bool ok = true;
            int asked = 0;
            for (int i = 0; ok && i < nblk; ++i) {
                const int st = i % XT_STAGES;
                if (i >= XT_STAGES) ok = warp_wait(&freed[st], ((i / XT_STAGES) - 1) & 1, abort, error_flag, 41);
                if (!ok) break;
                if (i * boxes - ids_from >= 32) { ids_from += 32; ids = ids_next; ids_next = ids_at(ids_from + 32); }
                const int id = __shfl_sync(0xffffffffu, ids, i * boxes + box - ids_from);
                // the box's first row among the cache's rows (past them: zeros)
                const int from_row = id < 0 ? arg.cache_rows : (int)((((unsigned)id * (unsigned)a.K + (unsigned)kh) << a.page_shift) + (unsigned)(((block0 + i) * XT_BN + box * rows) & (page - 1)));
                uint8_t* dst = (keys ? sK : sV) + st * XT_KV;
                // the box that the source ends in: its values by plain stores, zeros from there on
                const int tail = keys ? XT_BN : len - (block0 + i) * XT_BN, cut = tail < XT_BN ? tail / rows : boxes;
                const bool partial = cut < boxes && tail % rows != 0;
                if (partial) {
                    const bf16* src = cross_row<bf16>(a, a.v_cache, table, kh, (block0 + i) * XT_BN + cut * rows);
                    for (int x = lane; x < rows * NH * 8; x += 32) {
                        const int rw = x / (NH * 8), c = x % (NH * 8), at = cut * rows + rw;
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (at < tail && c * 8 < D) v = *reinterpret_cast<const uint4*>(src + (size_t)rw * D + c * 8);
                        *reinterpret_cast<uint4*>(dst + (c >> 3) * (XT_BN * 128) + at * 128 + (((c & 7) ^ (at & 7)) << 4)) = v;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (lane == 0) mbar_expect_tx(&full[st], (uint32_t)(XT_KV - (partial ? NH * rows * 128 : 0)));
                __syncwarp();
                if (loads && !(partial && box == cut)) tma_load_2d(dst + panel * (XT_BN * 128) + box * rows * 128, map, panel * 64, from_row, &full[st]);
                asked = i + 1;
            }
            // (what was asked for has to land before the block ends; where all went well the issuer has waited for it)
            if (!ok)
                for (int i = max(0, asked - XT_STAGES); i < asked; ++i) mbar_wait_warp(&full[i % XT_STAGES], (i / XT_STAGES) & 1);
        } else if (role == 6) {
            // ---- the issuer ----
            constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(XT_BN >> 3) << 17) | ((uint32_t)(XT_BM >> 4) << 24);
            constexpr uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(XT_BM >> 4) << 24);
            const uint32_t elected = elect_one(), tmem_s = warp_same(tmem_base), tmem_o = tmem_s + XT_O_COL;
            const int blocks = warp_same(nblk);
            const uint64_t qdesc = umma_desc(smem_u32(sQ));
            auto scores = [&](int i) {
                const int st = i % XT_STAGES;
                const uint64_t kdesc = umma_desc(smem_u32(sK) + st * XT_KV);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_bf16(tmem_s + (uint32_t)((i & 1) * XT_BN), qdesc + (uint32_t)((kk / 4) * (XT_BM * 128 >> 4) + 2 * (kk % 4)),
                              kdesc + (uint32_t)((kk / 4) * (XT_BN * 128 >> 4) + 2 * (kk % 4)), idesc_s, kk > 0 ? 1u : 0u, elected);
                umma_commit(&s_full[i & 1], elected);
                umma_commit(&k_free[st], elected);
            };
            bool ok = blocks > 0 && warp_wait(q_full, 0, abort, error_flag, 42);
            for (int i = 0; ok && i < min(2, blocks); ++i) {
                ok = warp_wait(&k_full[i % XT_STAGES], (i / XT_STAGES) & 1, abort, error_flag, 42);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                scores(i);
            }
            for (int i = 0; ok && i < blocks; ++i) {
                const int st = i % XT_STAGES, next = i + 2;
                const bool more = i + 2 < blocks;
                ok = warp_wait(&v_full[st], (i / XT_STAGES) & 1, abort, error_flag, 43);
                if (ok && more) ok = warp_wait(&k_full[next % XT_STAGES], (next / XT_STAGES) & 1, abort, error_flag, 45);
                // (The rows wait for few of o_done's phases, and a wait for a phase says nothing unless the one before it is known to be over; nothing orders the arrivals of two commits
                // on two barriers.  So each phase is seen here, before this block's weights are, which come later anyway: whoever sees the scores of block i knows that P V of
                // block i - 4 and of those ahead of it has arrived, and asks for i - 1 at the latest, four barriers in turn.)
                if (ok && i >= 2) ok = warp_wait(&o_done[(i - 2) & 3], ((i - 2) >> 2) & 1, abort, error_flag, 47);
                if (ok) ok = warp_wait(&p_full[i & 1], (i >> 1) & 1, abort, error_flag, 44);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t vdesc = umma_desc_mn(smem_u32(sV) + st * XT_KV, XT_BN * 128);
#pragma unroll
                for (int kk = 0; kk < XT_BN / 16; ++kk)
                    umma_bf16_tmem_a(tmem_o, tmem_s + (uint32_t)((i & 1) * XT_BN + kk * 8), vdesc + (uint32_t)(kk * (2048 >> 4)), idesc_pv, (i > 0 || kk > 0) ? 1u : 0u, elected);
                umma_commit(&o_done[i & 3], elected);
                umma_commit(&v_free[st], elected);
                if (more) scores(i + 2);                            // (S goes where P lies: the tensor core takes an issuer's products in their order)
            }
            if (!ok && blocks > 0) {                                // (and what was issued has to end)
                umma_commit(drained, elected);
                mbar_wait_warp(drained, 0);
            }
        }
    } else {
        // ---- the rows ----
        const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_col = lane_base + XT_O_COL;
        const float sl2 = a.scale * 1.4426950408889634f;
        // (rows that are not there or see nothing: their results are not looked at, so their scores need no mask)
        const int mask_from = range.y > range.x ? range.x : -0x40000000, mask_to = range.y > range.x ? range.y : 0x7fffffff;
        float m_used = -INFINITY, l_run = 0.0f;
        bool ok = true;
        for (int i = 0; i < nblk; ++i) {
            const uint32_t s_col = lane_base + (uint32_t)((i & 1) * XT_BN);
            ok = warp_wait(&s_full[i & 1], (i >> 1) & 1, abort, error_flag, 46);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float s[XT_BN];
            tmem_ld32_async(s_col, s);
            tmem_ld32_async(s_col + 32, s + 32);
            tmem_ld_wait(s);
            tmem_ld_wait(s + 32);
            const int key0 = (block0 + i) * XT_BN, from = mask_from - key0, to = mask_to - key0;
            if (__any_sync(0xffffffffu, from > 0 || to < XT_BN)) {
#pragma unroll
                for (int j = 0; j < XT_BN; ++j)
                    if (j < from || j >= to) s[j] = -INFINITY;
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < XT_BN; j += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) m4[e] = max3(m4[e], s[j + 2 * e], s[j + 2 * e + 1]);
            const float m_true = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
            float corr = 1.0f;
            const bool raise = m_true > m_used + 8.0f || (m_used == -INFINITY && m_true != -INFINITY);
            if (__any_sync(0xffffffffu, raise)) {
                if (raise) { corr = xt_exp2(m_used - m_true); m_used = m_true; }
                if (i > 0) {                                        // (P V of the blocks ahead has to be done)
                    ok = warp_wait(&o_done[(i - 1) & 3], ((i - 1) >> 2) & 1, abort, error_flag, 47);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        float o[16];
                        tmem_ld16(o_col + c * 16, o);
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] *= corr;
                        tmem_st16(o_col + c * 16, o);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
            }
            const float base = m_used == -INFINITY ? 0.0f : m_used;
            const uint64_t scale2 = pair_of(sl2, sl2), base2 = pair_of(-base, -base);
            uint64_t sum2[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < XT_BN / 32; ++c) {
                uint32_t packed[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint64_t x = fma_pair(pair_of(s[c * 32 + 2 * j], s[c * 32 + 2 * j + 1]), scale2, base2);
                    float p0, p1;
                    of_pair(x, p0, p1);
                    p0 = xt_exp2(p0); p1 = xt_exp2(p1);
                    sum2[j & 1] = add_pair(sum2[j & 1], pair_of(p0, p1));
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(packed[j]) : "f"(p1), "f"(p0));
                }
                tmem_st16_bits(s_col + c * 16, packed);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[i & 1]);
            float u0, u1;
            of_pair(add_pair(sum2[0], sum2[1]), u0, u1);
            l_run = l_run * corr + (u0 + u1);
        }
        if (nblk == 0) warp_wait(q_full, 0, abort, error_flag, 42);     // (nothing to do in this block of a cluster: what was asked for has to land all the same)
        if (ok && nblk > 0) ok = warp_wait(&o_done[(nblk - 1) & 3], ((nblk - 1) >> 2) & 1, abort, error_flag, 47);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float* sO = (float*)smem + (size_t)tid * XT_OLD;
        if (cluster > 1) {
            // the tile's memory is about to be written over: by now all products are done (this warp has seen it), and every warp of the rows says so
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        if (ok) {
            uint4* stage = reinterpret_cast<uint4*>(sQ);            // (the queries': the products are done)
            const bool sees = range.y > range.x;
            const float inv = 1.0f / l_run;
            const uint64_t inv2 = pair_of(inv, inv);
            uint64_t odd2 = 0;                                      // 0 times every result: NaN where one is not finite
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; ++c) {               // 64 columns at a time (of the last ones what there is: tensor memory behind them is this block's own)
                constexpr int MOST = D < 64 ? (D + 31) / 32 * 32 : 64;
                float o[MOST];
                if (nblk > 0) {
                    tmem_ld32_async(o_col + c * 64, o);
                    if (MOST > 32) tmem_ld32_async(o_col + c * 64 + 32, o + MOST - 32);
                    tmem_ld_wait(o);
                    if (MOST > 32) tmem_ld_wait(o + MOST - 32);
                } else {
#pragma unroll
                    for (int j = 0; j < MOST; ++j) o[j] = 0.0f;
                }
#pragma unroll
                for (int h = 0; h < MOST / 8; ++h) {
                    if (c * 64 + h * 8 >= D) continue;
                    if (cluster > 1) {
                        *reinterpret_cast<float4*>(sO + c * 64 + h * 8) = make_float4(o[8 * h], o[8 * h + 1], o[8 * h + 2], o[8 * h + 3]);
                        *reinterpret_cast<float4*>(sO + c * 64 + h * 8 + 4) = make_float4(o[8 * h + 4], o[8 * h + 5], o[8 * h + 6], o[8 * h + 7]);
                    } else {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint64_t xy = mul_pair(pair_of(o[8 * h + 2 * j], o[8 * h + 2 * j + 1]), inv2);
                            odd2 = fma_pair(xy, 0ull, odd2);
                            float x, y;
                            of_pair(xy, x, y);
                            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(y), "f"(x));
                        }
                        stage[XT_STAGED(tid, c * 8 + h)] = sees ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0u, 0u, 0u, 0u);
                    }
                }
            }
            bool odd = false;
            if (cluster == 1) {
                // a warp's rows out of shared memory, whole rows side by side (a thread its own row would touch 32 rows with every store), eight pieces a lane at a time
                __syncwarp();
                constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES, ROUNDS = (32 + AT_ONCE - 1) / AT_ONCE;
                const int piece = lane % PIECES;
#pragma unroll
                for (int r0 = 0; r0 < ROUNDS; r0 += 8) {
                    uint4 v[8];
                    int to[8];
#pragma unroll
                    for (int e = 0; e < 8 && r0 + e < ROUNDS; ++e) {
                        const int rw = (r0 + e) * AT_ONCE + lane / PIECES;
                        to[e] = lane < AT_ONCE * PIECES && rw < 32 ? s_to[warp * 32 + rw] : -1;
                        v[e] = stage[XT_STAGED(warp * 32 + min(rw, 31), piece)];
                    }
#pragma unroll
                    for (int e = 0; e < 8 && r0 + e < ROUNDS; ++e)
                        if (to[e] >= 0) reinterpret_cast<uint4*>(out0 + to[e])[piece] = v[e];
                }
                float z0, z1;
                of_pair(odd2, z0, z1);
                odd = mine && sees && z0 + z1 != 0.0f && cross_sum_speaks(l_run);
            }
            if (cluster > 1) { s_m[tid] = m_used; s_l[tid] = l_run; }
            if (a.spans != nullptr && cluster == 1) {
                unsigned which = __ballot_sync(0xffffffffu, odd);
                const int2 odd_values = which != 0 ? cross_odd_values<bf16, 1, true>(arg.a, kh, r, first_block * XT_BN, min(len, (first_block + blocks_all) * XT_BN)) : make_int2(0, 0);
                for (; which != 0; which &= which - 1) {
                    const int src = __ffs(which) - 1;
                    const int tok = __shfl_sync(0xffffffffu, my_tok, src), head = __shfl_sync(0xffffffffu, my_head, src);
                    const int2 rg = make_int2(__shfl_sync(0xffffffffu, range.x, src), __shfl_sync(0xffffffffu, range.y, src));
                    if (!cross_not_its_own(odd_values, rg)) continue;
                    __syncwarp();
                    cross_row_alone<bf16, 1, 4, true>(arg.a, tok0 + tok, head, r, rg);
                }
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 7) { __syncwarp(); tmem_free<false>(tmem_base, XT_TMEM); }
    if (cluster > 1) {
        cross_cluster_sync();
        // block `rank` finishes rows rank, rank + cluster, ...: a warp a row, four columns a lane
        const float* sO = (const float*)smem;
        bool looked = false;
        int2 odd_values = make_int2(0, 0);
        for (int done = rank + warp * cluster; done < XT_BM; done += (XT_THREADS / 32) * cluster) {
            const int to = s_to[done];
            if (to < 0) continue;
            float sum;
            const float factor = cross_factor<false>(&s_m[done], &s_l[done], cluster, sum);
            float4 v = cross_join4(sO + (size_t)done * XT_OLD + min(4 * lane, D - 4), factor, cluster);
            const int2 rg = s_range[done];
            const float inv = 1.0f / sum;
            v = rg.y > rg.x ? make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (4 * lane < D) {
                uint2 w;
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.x) : "f"(v.y), "f"(v.x));
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w.y) : "f"(v.w), "f"(v.z));
                reinterpret_cast<uint2*>(out0 + to)[lane] = w;
            }
            if (a.spans != nullptr && __any_sync(0xffffffffu, not_finite(v)) && cross_sum_speaks(sum)) {
                if (!looked) { looked = true; odd_values = cross_odd_values<bf16, 1, true>(arg.a, kh, r, first_block * XT_BN, min(len, (first_block + blocks_all) * XT_BN)); }
                if (cross_not_its_own(odd_values, rg)) { __syncwarp(); cross_row_alone<bf16, 1, 4, true>(arg.a, tok0 + to / (a.K * G * D), to / D % (a.K * G), r, rg); }
            }
        }
        cross_cluster_sync();                                       // (a block's shared memory is read until here)
    }
}

// ---- host side ----
static int map_rows(CUtensorMap* map, const void* base, uint64_t rows, uint32_t box_rows) {
    EncodeTiled enc = encode_tiled();
    if (enc == nullptr) return MB_ERR_BAD_SIZE;
    cuuint64_t dims[2] = {D, rows};
    cuuint64_t strides[1] = {D * 2};
    cuuint32_t box[2] = {64, box_rows};
    cuuint32_t elem[2] = {1, 1};
    const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : 1000 + (int)rc;
}
static int map_queries(CUtensorMap* map, const void* q, long long stride, int H, int tokens, int G, int per_tile) {
    EncodeTiled enc = encode_tiled();
    if (enc == nullptr) return MB_ERR_BAD_SIZE;
    cuuint64_t dims[3] = {D, (cuuint64_t)H, (cuuint64_t)tokens};
    cuuint64_t strides[2] = {D * 2, (cuuint64_t)stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)per_tile};
    cuuint32_t elem[3] = {1, 1, 1};
    const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? 0 : 1000 + (int)rc;
}

// Over how many blocks of a cluster the keys of a tile are cut: while there are fewer blocks than SMs, none with fewer than four blocks of keys.  (B200, heads of 128, 1, 2, 4
// and 8 blocks a tile: 32 tiles over 2,048 positions 25, 22, 16 and 17 us; 16 over 4,096 54, 34, 22 and 18; 80 over 4,096 51, 40, 46 and 53; 192 over 2,048 36, 50, 56, 94.)
static int choose_chunks(long long tiles, int longest) {
    const int keys = (longest + XT_BN - 1) / XT_BN;
    int c = 1;
    while (c < XT_MAX_CLUSTER && tiles * c * 2 <= XT_SMS + XT_SMS / 12 && keys >= 8 * c) c *= 2;
    return c;
}

// Pages of 16 to 128 positions; q, caches and out at 16 bytes, q_stride in whole 16-byte steps.
MB_API int mb_attention_cross_tc(const CrossCall* c, cudaStream_t s) {
    if (c->requests <= 0 || c->max_query <= 0) return 0;
    const long long cache_rows = c->cache_pages * c->K * c->page_size;
    if (!cross_call_fits(c) || c->d != D || c->dtype != MB_BF16 || c->page_size < 16 || c->page_size > 128 || c->H / c->K > XT_BM || cache_rows <= 0 || cache_rows > 0x7fffff00LL ||
        (((uintptr_t)c->q | (uintptr_t)c->k_cache | (uintptr_t)c->v_cache | (uintptr_t)c->out) & 15) != 0 || c->q_stride % 8 != 0 || (c->chunks != 0 && !chunks_fit(c->chunks)) ||
        (long long)c->H * D * 2 * XT_BM > 0x7fffffffLL)
        return MB_ERR_BAD_SIZE;
    const int G = c->H / c->K, per_tile = XT_BM / G;
    const CrossGrid grid = cross_grid(c, 1, per_tile);
    if (grid.blocks * c->K > 0x7fffffffLL) return MB_ERR_BAD_SIZE;
    static LaunchSmem allowed;
    int rc = allowed.allow(attention_cross_tc_kernel, XT_SMEM);
    if (rc != 0) return rc;
    const int chunks = c->chunks > 0 ? c->chunks : choose_chunks(grid.blocks * c->K, c->longest);
    CUtensorMap mq, mk, mv;
    const int box_rows = c->page_size < XT_BN ? c->page_size : XT_BN;
    if ((rc = map_queries(&mq, c->q, c->q_stride, c->H, c->tokens, G, per_tile)) != 0) return rc;
    if ((rc = map_rows(&mk, c->k_cache, (uint64_t)cache_rows, (uint32_t)box_rows)) != 0) return rc;
    if ((rc = map_rows(&mv, c->v_cache, (uint64_t)cache_rows, (uint32_t)box_rows)) != 0) return rc;
    const CrossTc arg = {cross_args(c), c->error_flag, c->first, c->requests, grid.max_tiles, (int)cache_rows};
    return launch_kernel(attention_cross_tc_kernel, dim3((unsigned)grid.blocks * c->K, 1, chunks), dim3(XT_THREADS), XT_SMEM, s, chunks, mq, mk, mv, arg);
}
