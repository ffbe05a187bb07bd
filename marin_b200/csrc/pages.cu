// A step's page bookkeeping on the device, from the requests' lengths before and after it (one launch, nothing read back):
//   request r holds pages(before[r]) pages and needs pages(after[r]) = ceil(after[r] / page_size).  Grown requests take pages, shrunk or
//   ended ones (after = 0) give theirs back; grown ones bring after - before new tokens.
//   The pages given back lie on top of the free list, in the order of requests and of their positions; pages are taken from its top in the same order:
//   take number i is entry pool - 1 - i of that stack, pool = count + given back.
// With the running sums over requests of new tokens, pages taken and pages given back, every output is worked out by itself: a token finds its
// request by bisection, its page in the block table or, if that page is one of this step's, in the stack; so there is no order between threads and no
// atomic, and the results are the same bits in every run.  Reads and writes are disjoint: the free list is read below `count` and written from there on,
// the block table is read where pages were held and written where they are new.
// Every block makes the running sums itself (R additions of three numbers, the lengths in shared memory: a second launch costs 2 to 3 us).
// Bound by latency: a launch, one round trip for the lengths, the sums' three rounds of shuffles, a bisection in shared memory, one round trip for a page.  Measured on
// B200, launches back to back: 8 requests 4.0 us, 256 with 24 prompts 4.6, 4,000 with 400 prompts and 100,000 new tokens 9.2 (12.0 with the lengths read again from memory by
// every token and three counts one after the other); the call takes the host 7.
#define MB_LIB "pages"
#define MB_LIB_ID 40
#include "common.cuh"
#include "launch.cuh"

#define PG_MAX_REQUESTS 8192
#define PG_PER (PG_MAX_REQUESTS / 1024)    // requests a thread at most
#define PG_LIMIT (1u << 30)        // sums stop here: what a launch can hold is less, and lengths nobody meant cannot wrap around

struct PageStep {
    const int* before;             // [R]
    const int* after;              // [R]
    int* table;                    // [R, columns]
    int* free;                     // [free_size], `count` of them filled
    const int* count;              // [1]
    int* left;                     // [2]: pages in the free list after the step; 0, or why nothing was done
    int* cu;                       // [R + 1]
    int* req;                      // [room] each
    int* pos;
    int* slots;
    int R, columns, free_size, shift, room;
};

__device__ __forceinline__ unsigned capped(unsigned v) { return v < PG_LIMIT ? v : PG_LIMIT; }
__device__ __forceinline__ int pages_for(int tokens, int shift) { return (int)(((unsigned)tokens + (1u << shift) - 1u) >> shift); }

// One request's new tokens, pages taken and pages given back, added to the sums.
__device__ __forceinline__ void add_request(unsigned* sum, int before, int after, int shift) {
    const int held = pages_for(before, shift), wants = pages_for(after, shift);
    sum[0] = capped(sum[0] + (unsigned)max(0, min(after - before, (int)PG_LIMIT)));
    sum[1] = capped(sum[1] + (unsigned)max(0, wants - held));
    sum[2] = capped(sum[2] + (unsigned)max(0, held - wants));
}

// The last r with upto[r] <= x (upto[0] = 0, not decreasing, x < upto[R]).
__device__ __forceinline__ int owner_of(const unsigned* upto, int R, unsigned x) {
    int lo = 0, hi = R;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (upto[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(1024) page_step_kernel(PageStep p) {
    extern __shared__ __align__(16) unsigned pg_sums[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const int per = max(4, ((p.R + threads - 1) / threads + 3) & ~3), padded = (p.R + 4) & ~3;       // requests a thread, side by side, in whole 16-byte steps; room for the sums' last
    int* before = reinterpret_cast<int*>(pg_sums);                  // [padded] each
    int* after = before + padded;
    unsigned* upto_new = reinterpret_cast<unsigned*>(after + padded);
    unsigned* upto_taken = upto_new + padded;
    unsigned* upto_back = upto_taken + padded;
    __shared__ unsigned warp_total[3][32];
    PDL_ENTER();
    p.before = pdl_fresh(p.before); p.after = pdl_fresh(p.after); p.table = pdl_fresh(p.table); p.free = pdl_fresh(p.free); p.count = pdl_fresh(p.count);
    const int count = p.count[0];
    int bad = 0;
    for (int r = tid; r < padded; r += threads) {
        const int b = r < p.R ? p.before[r] : 0, a = r < p.R ? p.after[r] : 0;
        bad |= a < 0 || b < 0 || pages_for(a, p.shift) > p.columns || pages_for(b, p.shift) > p.columns;
        before[r] = b; after[r] = a;
    }
    bad = __syncthreads_or(bad);
    const int first = tid * per;
    int b[PG_PER], a[PG_PER];
    unsigned upto[3] = {0u, 0u, 0u};                                // of the threads ahead of this one
    if (!bad) {
        unsigned sum[3] = {0u, 0u, 0u};
#pragma unroll
        for (int k = 0; k < PG_PER; k += 4) {
            int4 bv = make_int4(0, 0, 0, 0), av = bv;
            if (k < per && first + k < padded) { bv = *reinterpret_cast<const int4*>(before + first + k); av = *reinterpret_cast<const int4*>(after + first + k); }
            b[k] = bv.x; b[k + 1] = bv.y; b[k + 2] = bv.z; b[k + 3] = bv.w;
            a[k] = av.x; a[k + 1] = av.y; a[k + 2] = av.z; a[k + 3] = av.w;
        }
#pragma unroll
        for (int k = 0; k < PG_PER; ++k) add_request(sum, b[k], a[k], p.shift);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            unsigned v = sum[k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned other = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v = capped(v + other);
            }
            if (lane == 31) warp_total[k][warp] = v;
            const unsigned ahead = __shfl_up_sync(0xffffffffu, v, 1);
            upto[k] = lane == 0 ? 0u : ahead;
        }
    }
    __syncthreads();
    if (!bad) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            unsigned v = lane < (threads >> 5) ? warp_total[k][lane] : 0u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned other = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v = capped(v + other);
            }
            const unsigned ahead = __shfl_sync(0xffffffffu, v, (warp + 31) & 31);
            if (warp > 0) upto[k] = capped(upto[k] + ahead);
        }
#pragma unroll
        for (int k = 0; k < PG_PER; ++k) {
            const int r = first + k;
            if (k < per && r < p.R) { upto_new[r] = upto[0]; upto_taken[r] = upto[1]; upto_back[r] = upto[2]; }
            add_request(upto, b[k], a[k], p.shift);
        }
        // (whoever has the last request has all of them now: places behind it are zeros)
        if (first < p.R && first + per >= p.R) { upto_new[p.R] = upto[0]; upto_taken[p.R] = upto[1]; upto_back[p.R] = upto[2]; }
    }
    __syncthreads();
    unsigned n_new = 0, n_taken = 0, n_back = 0;
    int status = 3;
    if (!bad) {
        n_new = upto_new[p.R]; n_taken = upto_taken[p.R]; n_back = upto_back[p.R];
        status = n_new > (unsigned)p.room ? 2
                 : count < 0 || count > p.free_size ? 4
                 : n_taken > (unsigned)count + n_back ? 1
                 : (unsigned)count + n_back - n_taken > (unsigned)p.free_size ? 4 : 0;
    }
    const int at = blockIdx.x * threads + tid, stride = gridDim.x * threads;
    if (at == 0) {
        p.left[0] = status == 0 ? (int)((unsigned)count + n_back - n_taken) : count;
        p.left[1] = status;
    }
    if (status != 0) {
        for (int r = at; r <= p.R; r += stride) p.cu[r] = 0;
        for (int t = at; t < p.room; t += stride) { p.req[t] = 0; p.pos[t] = 0; p.slots[t] = -1; }
        return;
    }
    const unsigned pool = (unsigned)count + n_back;
    // page `i` of the stack: what the free list held, and on top of it what this step gives back
    auto stacked = [&](unsigned i) -> int {
        if (i < (unsigned)count) return p.free[i];
        const unsigned k = i - (unsigned)count;
        const int r = owner_of(upto_back, p.R, k);
        return p.table[(size_t)r * p.columns + pages_for(after[r], p.shift) + (int)(k - upto_back[r])];
    };
    for (int r = at; r <= p.R; r += stride) p.cu[r] = (int)upto_new[r];
    // tokens, pages taken and pages laid on the free list, one after the other in one count: a thread has one of them at most, as a rule
    const unsigned kept = n_back > n_taken ? n_back - n_taken : 0u, all = (unsigned)p.room + n_taken + kept;
    for (unsigned x = at; x < all; x += stride) {
        if (x < (unsigned)p.room) {
            int r = 0, position = 0, slot = -1;
            if (x < n_new) {
                r = owner_of(upto_new, p.R, x);
                const int had = before[r], held = pages_for(had, p.shift);
                position = had + (int)(x - upto_new[r]);
                const int column = position >> p.shift;
                const int page = column < held ? p.table[(size_t)r * p.columns + column] : stacked(pool - 1u - (upto_taken[r] + (unsigned)(column - held)));
                slot = (page << p.shift) + (position & ((1 << p.shift) - 1));
            }
            p.req[x] = r; p.pos[x] = position; p.slots[x] = slot;
        } else if (x < (unsigned)p.room + n_taken) {
            const unsigned i = x - (unsigned)p.room;
            const int r = owner_of(upto_taken, p.R, i);
            p.table[(size_t)r * p.columns + pages_for(before[r], p.shift) + (int)(i - upto_taken[r])] = stacked(pool - 1u - i);
        } else {
            const unsigned i = (unsigned)count + (x - (unsigned)p.room - n_taken);
            p.free[i] = stacked(i);
        }
    }
}

static bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// before, after [R], table [R, columns], free [free_size], count [1], left [2], cu [R + 1], req, pos, slots [room]: int32.  page_size: a power of two.
// left[1]: 0; 1: the free list runs out of pages; 2: more new tokens than `room`; 3: a length is negative or needs more pages than a row of the table
// has; 4: the free list cannot hold what is given back (or `count` is none of its lengths).  Where it is not 0 nothing is taken or given back.
struct PageStepCall {              // (in one piece: a caller in Python pays for every argument)
    const int *before, *after;
    int *table, *free;
    const int* count;
    int *left, *cu, *req, *pos, *slots;
    int R, columns, free_size, page_size, room;
};

MB_API int mb_page_step(const PageStepCall* c, cudaStream_t s) {
    const int R = c->R, columns = c->columns, free_size = c->free_size, page_size = c->page_size, room = c->room;
    if (R <= 0 || R > PG_MAX_REQUESTS || columns <= 0 || (long long)R * columns >= PG_LIMIT || free_size < 0 || free_size >= (int)PG_LIMIT || room < 0 ||
        room >= (int)PG_LIMIT || page_size <= 0 || (page_size & (page_size - 1)) != 0)
        return MB_ERR_BAD_SIZE;
    // what every block reads must not be what another has written by then
    const void* part[] = {c->before, c->after, c->count, c->table, c->free, c->left, c->cu, c->req, c->pos, c->slots};
    const size_t n[] = {(size_t)R, (size_t)R, 1, (size_t)R * columns, (size_t)free_size, 2, (size_t)R + 1, (size_t)room, (size_t)room, (size_t)room};
    for (int i = 0; i < 10; ++i)
        for (int j = i + 1; j < 10; ++j)
            if (j >= 3 && overlap(part[i], n[i] * 4, part[j], n[j] * 4)) return MB_ERR_BAD_SIZE;
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    const int threads = R <= 256 ? 256 : 1024;
    // (pages given back are the device's to know: room for four a request)
    const long long items = (long long)room + room / 16 + 4LL * R;
    const int blocks = (int)max(1LL, min(148LL, (items + threads - 1) / threads));
    const size_t smem = 5 * (((size_t)R + 4) & ~(size_t)3) * sizeof(unsigned);
    static LaunchSmem allowed;
    const int rc = allowed.allow(page_step_kernel, 5 * (PG_MAX_REQUESTS + 4) * sizeof(unsigned));
    if (rc != 0) return rc;
    const PageStep p = {c->before, c->after, c->table, c->free, c->count, c->left, c->cu, c->req, c->pos, c->slots, R, columns, free_size, shift, room};
    return launch_kernel(page_step_kernel, dim3(blocks), dim3(threads), smem, s, 0, p);
}
