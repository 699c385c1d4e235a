// One step's bookkeeping of a paged key-value cache, in one launch: which requests get their new tokens, which pages they
// take off the stack of free ones, and in which slot of the cache each token goes.
//
//   held_r = ceil(len_r / P), need_r = ceil((len_r + new_r) / P) - held_r          (P tokens to a page)
//   first_r = sum of need over the requests before r: request r takes the pages first_r .. first_r + need_r - 1 from the top
//   slot of its j-th token = table[r][(len_r + j) / P] * P + (len_r + j) % P
//
// A few integers per request: bound by latency (the launch, a load, a prefix sum over the requests, the dependent load of a
// page).  Every CTA makes the prefix sums for itself, in shared memory, and the work that follows is dealt out by pages and by
// rows (found again by binary search), not by requests: one long prompt is shared out as evenly as many short ones.  A
// decode step fits one CTA; many rows are written by a cluster of eight, whose barriers keep the order of the phases.
#include "paged_plan.h"

#include <limits.h>

#include "dlr_b200.h"
#include "ptx.cuh"

namespace dlr {

namespace {

constexpr int kThreadsP = 512;
constexpr int kWarpsP = kThreadsP / 32;
constexpr int kClusterP = 8;
// Rows above which eight CTAs beat one (us, 16 requests): 2048 rows 4.7 and 5.0, 1024 rows 4.7 and 4.2, 16384 rows 4.6 and 14.1,
// 128000 rows (64 requests) 8.8 and 89; 4096 requests with a row each 17 and 23.
constexpr int kClusterRows = 1536;

// inclusive sums over the CTA's threads; `total` is the sum of all
struct Sums {
    long long pages, rows;
};

__device__ Sums scan(Sums v, Sums* scratch, Sums* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long p = __shfl_up_sync(~0u, v.pages, o), r = __shfl_up_sync(~0u, v.rows, o);
        if (lane >= o) {
            v.pages += p;
            v.rows += r;
        }
    }
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    Sums before{0, 0}, all{0, 0};
#pragma unroll
    for (int w = 0; w < kWarpsP; ++w) {
        const Sums s = scratch[w];
        if (w < warp) {
            before.pages += s.pages;
            before.rows += s.rows;
        }
        all.pages += s.pages;
        all.rows += s.rows;
    }
    __syncthreads();
    v.pages += before.pages;
    v.rows += before.rows;
    *total = all;
    return v;
}

__device__ __forceinline__ int clamped(long long v) { return v > INT_MAX ? INT_MAX : int(v); }

// the last of first[0..n) that is not above a (first[0] = 0 <= a)
__device__ __forceinline__ int owner(const int* first, int n, int a) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= a) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <bool CLUSTER>
__device__ __forceinline__ void barrier() {
    if constexpr (CLUSTER) {
        __syncwarp();                        // (the barrier is one of whole warps)
        cluster_arrive_release();
        cluster_wait_acquire();
    } else {
        __syncthreads();
    }
}

template <bool CLUSTER>
__global__ void __launch_bounds__(kThreadsP) plan_kernel(const PlanArgs a) {
    extern __shared__ int memory[];
    __shared__ Sums scratch[kWarpsP];
    __shared__ int used;
    const int R = a.requests, rank = CLUSTER ? int(cluster_ctarank()) : 0, ctas = CLUSTER ? kClusterP : 1;
    const int worker = rank * kThreadsP + threadIdx.x, workers = ctas * kThreadsP;
    int* const old_length = memory;            // tokens held, once the finished requests are gone
    int* const added = old_length + R;         // tokens that the request gets
    int* const first = added + R;              // pages asked for by the requests before (and, at first, pages given back)
    int* const start = first + R;              // rows of the requests before, where there is no fixed width
    const long long page = 1ll << a.page_shift, capacity = min((long long)a.columns << a.page_shift, (long long)INT_MAX);
    auto pages_of = [&](long long tokens) { return (tokens + page - 1) >> a.page_shift; };
    auto held = [&](int r) { return min(max((long long)a.lengths[r], 0ll), capacity); };
    const int n_free = min(max(*a.n_free, 0), a.pool);
    int available = n_free;
    if (threadIdx.x == 0) used = 0;

    if (a.finished) {
        Sums base{0, 0}, total;
        for (int r0 = 0; r0 < R; r0 += kThreadsP) {
            const int r = r0 + int(threadIdx.x);
            const long long mine = r < R && a.finished[r] ? pages_of(held(r)) : 0;
            const Sums s = scan({mine, 0}, scratch, &total);
            if (r < R) first[r] = clamped(base.pages + s.pages - mine);
            base.pages += total.pages;
        }
        __syncthreads();
        const int back = int(min(base.pages, (long long)(a.pool - n_free)));     // (no more than the stack has room for)
        for (int i = worker; i < back; i += workers) {
            const int r = owner(first, R, i);
            a.free_pages[n_free + i] = a.block_table[r * a.table_stride + (i - first[r])];
        }
        available += back;
        barrier<CLUSTER>();           // every returned page is on the stack, and was read before its entry is written again
    }

    Sums base{0, 0}, total;
    for (int r0 = 0; r0 < R; r0 += kThreadsP) {
        const int r = r0 + int(threadIdx.x);
        long long old = 0, wanted = 0, need = 0;
        if (r < R) {
            old = a.finished && a.finished[r] ? 0 : held(r);
            wanted = max(a.new_tokens[r], 0);
            if (old + wanted <= capacity && (a.width == 0 || wanted <= a.width)) need = pages_of(old + wanted) - pages_of(old);
        }
        const Sums s = scan({need, wanted}, scratch, &total);
        if (r < R) {
            const long long last = base.pages + s.pages, last_row = base.rows + s.rows;
            const bool fits = old + wanted <= capacity && (a.width ? wanted <= a.width : last_row <= a.rows);
            const bool granted = fits && (need == 0 || last <= available);
            old_length[r] = int(old);
            added[r] = granted ? int(wanted) : 0;
            first[r] = clamped(last - need);
            start[r] = a.width ? clamped((long long)r * a.width) : clamped(last_row - wanted);
            if (granted && need > 0) atomicMax(&used, int(last));
        }
        base.pages += total.pages;
        base.rows += total.rows;
    }
    __syncthreads();

    // page i from the top of the stack goes to the request that asked for the i-th
    const int taken = int(min(base.pages, (long long)available));
    for (int i = worker; i < taken; i += workers) {
        const int r = owner(first, R, i);
        if (added[r] > 0)
            a.block_table[r * a.table_stride + pages_of(old_length[r]) + (i - first[r])] = __ldcg(a.free_pages + (available - 1 - i));
    }
    barrier<CLUSTER>();               // the tables are complete, and every CTA has read the lengths and the stack's count

    // Rows: where there are many, four neighbouring ones to a thread, found once, walked from there, stored as one.  (128000 rows:
    // 9 us, 15 with a row at a time.)
    constexpr int kEach = CLUSTER ? 4 : 1;
    const int mask = int(page) - 1;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15u) == 0;
    auto slot_at = [&](int r, int position) {
        const int at = a.block_table[r * a.table_stride + (position >> a.page_shift)];
        return at >= 0 && at <= INT_MAX >> a.page_shift ? (at << a.page_shift) + (position & mask) : -1;
    };
    for (int i = kEach * worker; i < a.rows; i += kEach * workers) {
        int slot[kEach], position[kEach];
        int r = R == 0 ? 0 : a.width ? i / a.width : owner(start, R, i);
        const int j0 = r < R ? i - start[r] : 0, here = r < R ? added[r] - j0 : 0;       // tokens of this request from row i on
        const int first_position = r < R ? old_length[r] + j0 : 0;
        if (here >= kEach && (first_position & mask) + kEach <= mask + 1) {              // all on one page
            const int first_slot = slot_at(r, first_position);
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                position[k] = first_position + k;
                slot[k] = first_slot < 0 ? -1 : first_slot + k;
            }
        } else {
            const bool behind = here <= 0 && (r + 1 >= R || start[r + 1] >= i + kEach);  // none has a token
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                slot[k] = -1;
                position[k] = 0;
                if (behind) continue;
                while (kEach > 1 && r + 1 < R && start[r + 1] <= i + k) ++r;
                const int j = r < R ? i + k - start[r] : 0;
                if (r < R && j < added[r]) {
                    position[k] = old_length[r] + j;
                    slot[k] = slot_at(r, position[k]);
                }
            }
        }
        if (kEach == 4 && wide && i + 4 <= a.rows) {
            *reinterpret_cast<int4*>(a.slots + i) = make_int4(slot[0], slot[1 % kEach], slot[2 % kEach], slot[3 % kEach]);
            *reinterpret_cast<int4*>(a.positions + i) = make_int4(position[0], position[1 % kEach], position[2 % kEach], position[3 % kEach]);
        } else {
#pragma unroll
            for (int k = 0; k < kEach; ++k)
                if (i + k < a.rows) {
                    a.slots[i + k] = slot[k];
                    a.positions[i + k] = position[k];
                }
        }
    }
    if (rank != 0) return;
    for (int r = threadIdx.x; r < R; r += kThreadsP) {
        a.lengths_out[r] = old_length[r] + added[r];
        a.starts[r] = start[r];
    }
    if (threadIdx.x == 0) {
        a.starts[R] = a.width ? clamped((long long)R * a.width) : clamped(base.rows);
        *a.n_free_out = available - used;
    }
}

}  // namespace

cudaError_t paged_plan(const PlanArgs& a, int smem_optin, cudaStream_t stream) {
    const bool cluster = a.rows > kClusterRows;
    const size_t smem = size_t(a.requests) * 4 * sizeof(int);
    auto kern = cluster ? plan_kernel<true> : plan_kernel<false>;
    if (smem > 40 * 1024) {
        // the most that any call takes: a call of fewer requests in another thread, between this and the launch, would lower it
        constexpr int kMost = DLRB200_MAX_PLAN_REQUESTS * 4 * int(sizeof(int));
        if (smem > size_t(kMost) || kMost + 1024 > smem_optin) return cudaErrorInvalidValue;
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {unsigned(kClusterP), 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster ? kClusterP : 1);
    cfg.blockDim = dim3(kThreadsP);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace dlr
