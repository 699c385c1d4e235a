// Attention of one new token per request over a paged key-value cache:
//
//   o_h = sum_j softmax_j(scale * q_h . k_j) v_j     over the tokens j of the request; zeros where there are none
//
// Bound by memory: the keys and values of a request are read once for up to 16 query heads that share them (more: once for each 16),
// and each value read serves one multiply-add for each of these heads, far below what the tensor cores give.
//
// Split.  The work is a list of tiles of 64 tokens: request by request, key-value head by key-value head.  It is cut into
// equal runs, a few for each CTA, wherever the cuts fall: short requests share a CTA, a long one is spread over all of them, ragged
// batches stay balanced, and the host needs to know no length.  A CTA works through its run segment by segment (the tiles of
// one request and head).  What is cut is joined by a second, small kernel from partial results in fp32, in the order of the
// tokens, so that results repeat bit for bit; what is whole is finished by its CTA.  Where the table holds short contexts only, a
// cluster takes each head's tokens instead and joins them through distributed shared memory: one launch.
//
// A warp takes 16 tokens of a tile at a time, on its own: it copies their keys and their values to its own ring in shared memory
// (cp.async, rows padded by 16 bytes so that ldmatrix meets no bank twice), multiplies with mma.sync, and keeps maximum, sum and
// output of its tokens in registers; the warps of a CTA are joined at the end of a segment.  Scores are (heads x tokens), the
// output is turned round, (values x heads): the scores' registers then are the second product's operand as they are, and the
// output of eight heads takes half the registers that 16 rows would.  A softmax weight enters that product as a sum of 16-bit terms,
// three in bf16 (all 24 bits of it; two, 16 bits, where more than eight heads share keys), two in fp16 (22 bits).
#include "paged_attention.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace dlr {

namespace {

constexpr int kWarpsA = 4;
constexpr int kThreadsA = 32 * kWarpsA;
constexpr int kWarpsJ = 8;                       // of the joining kernel
constexpr int kThreadsJ = 32 * kWarpsJ;
constexpr int kMostHeads = 64;                   // of a CTA of it
constexpr int kUnit = 16;                        // tokens of a warp's step
constexpr int kTile = kUnit * kWarpsA;           // tokens of a tile
// CTAs of an SM for heads of `dim`, nt groups of eight sharing keys: as many as registers and shared memory allow.  More warps
// count for more than more copies in flight: a warp's step is a chain of dependent instructions (460 MB, us: 6 heads of 128 with
// 3 CTAs of 3 halves 80, of 4 halves 81, 2 CTAs of 5 or 6 halves 82; 3 heads of 256 with 2 CTAs of 2 halves 82, of 3 halves 93, one CTA
// of 4 86).
constexpr int ctas_per_sm(int dim, int nt) { return dim == 64 ? 4 : dim == 96 ? (nt == 1 ? 4 : 3) : dim == 128 ? 3 : 2; }
constexpr int kMostCtasPerSm = 4;
// Runs for each resident CTA, and tiles of a run below which there is one for each.  Measured with 1 / 2 / 4 / 6 runs (kernel and
// join, us): 64 ragged requests of up to 8000 tokens, 8 heads of 128: 173 / 171 / 167 / 166; one of 131072: 93 / 93 / 93 / 93; 200
// of up to 1500, 12 heads of 64: 92 / 94 / 94 / 94 with at least 32 tiles, 84 with 8 (32 was chosen before the output was turned
// round, when it took 83); heads of 128 with at least 8: as with 16.
constexpr int kWaves = 4;
constexpr int least_run(int dim) { return dim == 64 ? 32 : 16; }
constexpr int kMostShares = 8;                   // CTAs of a cluster
// Tiles of a share up to which a cluster for each segment is taken instead of the runs and their join, by what the table could
// hold (the host knows no lengths).  us, runs / clusters, contexts of one length, then ragged ones, 8 heads of 128, up to 40 caches
// in turn (400 MB, above what L2 holds, but for the first case): 1 request of 513 tokens, 2 tiles: 7.1 / 5.3; 8 of 768, 2 tiles: 11.2 /
// 7.9, 10.1 / 6.8; 8 of 2000, 8 tiles: 19.2 / 13.7, 14.4 / 11.3; 32 of 768, 12 tiles: 31.9 / 18.4, 24.0 / 14.8; 256 of 700, 11 tiles:
// 123 / 115, 73 / 63.  Above: 64 of 1000, 16 tiles: 48 / 56, 29 / 28.
constexpr int kShort = 12;
constexpr int kMostSms = 160;
constexpr int kMostParts = kMostCtasPerSm * kMostSms * kWaves;
constexpr float kLog2e = 1.4426950408889634f;
// What the weights (1 at most) are multiplied by before they are split in terms; the output is brought back at the end.  bf16 reaches as
// far down as fp32.  fp16 ends 2^-24 below 1, which a long tail of tokens beside one large weight would feel: with 2^15 a weight is
// right to 2^-16 of itself down to 2^-24 of the largest one, to 2^-40 of the largest one down to 2^-39 of it, and to 2^-38 below.
template <typename T>
constexpr float kWeightUp = __is_same(T, __half) ? 32768.f : 1.f;
// Terms of a weight: those of fp16, and of bf16 for NT groups of eight heads that share keys.
template <typename T, int NT>
constexpr int kTerms = __is_same(T, __half) || NT > 1 ? 2 : 3;
template <typename T>
constexpr float kLeastTerm = __is_same(T, __half) ? 0x1p-24f : 0x1p-126f;

template <int D, int NT>
struct Shape {
    static constexpr int kRow = D * 2 + 16;                        // bytes of a row in shared memory
    static constexpr int kHalf = kUnit * kRow;                     // keys (or values) of a step
    static constexpr int kHalves = D <= 128 ? 3 : 2;               // of a warp's ring
    static constexpr int kRing = kWarpsA * kHalves * kHalf;
    static constexpr int kRows = 8 * NT;                           // query heads of a segment
    static constexpr int kJoinRow = D + 4;                         // floats; the padding keeps banks apart
    static constexpr int kJoin = kWarpsA * kRows * kJoinRow * 4;   // output of every warp; its maxima and sums lie behind
    static constexpr int kCtasPerSm = ctas_per_sm(D, NT);
    // the join has memory of its own where there is room, so that the next segment's copies can start before it
    static constexpr int kMl = kWarpsA * kRows * 8;
    static constexpr bool kApart = kRing + kJoin + kMl + 1280 <= 228 * 1024 / kCtasPerSm;
    static constexpr int kJoinAt = kApart ? kRing : 0, kMlAt = kApart ? kRing + kJoin : kRing > kJoin ? kRing : kJoin;
    static constexpr int kSmem = kMlAt + kMl;
    static constexpr int kPart = kRows * (D + 2);                  // floats of a partial result: output, maxima, sums
};

// (the hint: keys and values go first from L2, and leave the partial results there)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes, uint64_t hint) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(hint) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __half)) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// two values in 16 bits, rounded toward zero
template <typename T>
__device__ __forceinline__ uint32_t toward_zero2(float x, float y) {
    uint32_t v;
    if constexpr (__is_same(T, __half)) asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(y), "f"(x));
    else v = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    return v;
}

template <typename T>
__device__ __forceinline__ float2 floats2(uint32_t v) {
    if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return make_float2(bf16lo_to_f(v), bf16hi_to_f(v));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (__is_same(T, __half)) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return pack_bf16x2(x, y);
    }
}

// Two weights as sums of 16-bit terms.  All terms of a weight above 0 are above 0: a term that is zero or negative would turn an
// infinite value into NaN or the other infinity, by the weight's bits.  Hence the rounding toward zero; the last term takes what is left.
// (Outputs are 1e-4 away from those of fp32 weights with two terms of bf16, 5e-5 with three, which is what sums in another order
// do; both far below their rounding to bf16.  us with two signed terms / three: 64 ragged requests of up to 8000 tokens, 4 heads of
// 128 to a key head 164.4 / 165.1; one of 131072, 8 heads to a key head 91.8 / 93.0.  460 MB of ragged requests, 12 heads to a key
// head, two signed terms / two / three: heads of 64 130 / 131 / 145, of 128 90 / 90 / 96, of 256 135 / 135 / 146.  Two signed terms,
// and the tokens once more where an output is not finite, in these five cases: 166.3, 93.0, 139, 91.5, 137.)
template <typename T, int TERMS>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&term)[TERMS]) {
    const float least_x = x > 0.f ? kLeastTerm<T> : 0.f, least_y = y > 0.f ? kLeastTerm<T> : 0.f;
    if constexpr (__is_same(T, __half)) {      // (half of the least term less: together the two are off by as much up as down)
        term[0] = toward_zero2<T>(fmaxf(x - kLeastTerm<T> / 2, least_x), fmaxf(y - kLeastTerm<T> / 2, least_y));
    } else {
        term[0] = toward_zero2<T>(x, y);
    }
#pragma unroll
    for (int i = 1; i < TERMS; ++i) {
        const float2 before = floats2<T>(term[i - 1]);
        x = fmaxf(x - before.x, least_x);
        y = fmaxf(y - before.y, least_y);
        term[i] = i + 1 < TERMS ? toward_zero2<T>(x, y) : pack2<T>(x, y);
    }
}

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr_cluster) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr_cluster) : "memory");
    return v;
}

__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(~0u, v, 1));
    return fmaxf(v, __shfl_xor_sync(~0u, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(~0u, v, 1);
    return v + __shfl_xor_sync(~0u, v, 2);
}

constexpr int kEach = 8;                         // requests that a thread counts at a time

// Tokens and tiles of a request.
struct Geometry {
    const int* lengths;
    int requests, segments;              // segments of a request: key-value heads x groups of query heads
    long long capacity;

    __device__ __forceinline__ int tokens(int r) const {
        const long long n = lengths[r];
        return int(n < 0 ? 0 : n > capacity ? capacity : n);
    }
    // tiles of the requests r, r + 1, ... that a thread counts, and all of them (below 2^31 for each: host check)
    __device__ __forceinline__ long long some(int r, int (&tiles)[kEach]) const {
        long long sum = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            tiles[k] = r + k < requests ? (tokens(r + k) + kTile - 1) / kTile * segments : 0;
            sum += tiles[k];
        }
        return sum;
    }
};

// Sums of v over the warps' lanes: what lies before this thread, and all.
template <int WARPS>
__device__ __forceinline__ long long scan_tiles(long long v, long long* scratch, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += scratch[w];
        all += scratch[w];
    }
    __syncthreads();
    *total = all;
    return before + sum - v;
}

// How the tiles are cut: into as many runs as CTAs are resident, or several times as many while runs stay long, so that SMs
// that get more of the memory's bandwidth than others take more of them.
struct Cut {
    int resident, waves, least;          // CTAs, runs for each of them at most, tiles of a run if there is more than one for each

    __device__ __forceinline__ long long run(long long total) const {
        const long long fit = total / ((long long)resident * least);
        const long long runs = (long long)resident * (fit < 1 ? 1 : fit < waves ? fit : waves), even = (total + runs - 1) / runs;
        return even < 1 ? 1 : even;
    }
};

// The request that holds tile `at`, and the tiles before it.
struct Place {
    int request;
    long long before;
};

// SHARED: a cluster of `shares` CTAs to each segment instead, which take equal shares of its tiles and are joined through
// distributed shared memory (short contexts, where a second launch would cost as much as the work).
template <typename T, int D, int NT, bool SHARED>
__global__ void __launch_bounds__(kThreadsA, Shape<D, NT>::kCtasPerSm) paged_attention_kernel(const __grid_constant__ PagedAttention p, int groups, const Cut cut, int shares) {
    using S = Shape<D, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long scratch[kWarpsA];
    __shared__ Place place;
    __shared__ float2 share_ml[S::kRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group_size = p.heads / p.kv_heads;
    const Geometry geo{p.lengths, p.requests, p.kv_heads * groups, (long long)p.columns << p.page_shift};

    long long run = 0, at = 0, end = 0, before = 0;
    int request = 0;
    if constexpr (!SHARED) {
        asm volatile("griddepcontrol.launch_dependents;");
        // all tiles, and the request in which this CTA's run begins
        long long total = 0;
        int mine[kEach];
        for (int r0 = 0; r0 < p.requests; r0 += kThreadsA * kEach) {
            long long here;
            before = total + scan_tiles<kWarpsA>(geo.some(r0 + int(threadIdx.x) * kEach, mine), scratch, &here);
            total += here;
        }
        run = cut.run(total);
        at = run * blockIdx.x;
        end = at + run < total ? at + run : total;
        // requests without tokens belong to no tile: their zeros are written by the CTAs in turn
        for (int r = blockIdx.x; r < p.requests; r += gridDim.x)
            if (geo.tokens(r) == 0)
                for (int i = threadIdx.x; i < p.heads * D / 2; i += kThreadsA)
                    reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + int64_t(r) * p.heads * D)[i] = 0;
        if (at >= end) return;
        auto find = [&](int r, long long before) {
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                if (at >= before && at < before + mine[k]) place = {r + k, before};
                before += mine[k];
            }
        };
        if (p.requests <= kThreadsA * kEach) {
            find(int(threadIdx.x) * kEach, before);
        } else {
            long long base = 0;
            for (int r0 = 0; r0 < p.requests; r0 += kThreadsA * kEach) {
                const int r = r0 + int(threadIdx.x) * kEach;
                long long here;
                before = base + scan_tiles<kWarpsA>(geo.some(r, mine), scratch, &here);
                find(r, before);
                base += here;
            }
        }
        __syncthreads();
        request = place.request;
        before = place.before;
    }

    const uint32_t ring = smem_u32(smem) + warp * (S::kHalves * S::kHalf);
    float* const join = reinterpret_cast<float*>(smem + S::kJoinAt);
    float2* const join_ml = reinterpret_cast<float2*>(smem + S::kMlAt);
    const float scale = p.scale * kLog2e;
    const uint64_t hint = l2_policy_evict_first();

    // The run's next segment, as far as it lies in the run; none: 0 tokens.
    struct Piece {
        int request, tokens, segment, tile0, tile1, seg_tiles;
        bool opens;                             // it is the run's first
    };
    auto next_piece = [&]() {
        Piece a{};
        while (at < end) {
            a.tokens = geo.tokens(request);
            a.seg_tiles = (a.tokens + kTile - 1) / kTile;
            const long long behind = before + (long long)a.seg_tiles * geo.segments;
            if (at < behind) {
                a.request = request;
                a.segment = int(unsigned(at - before) / unsigned(a.seg_tiles));      // (below 2^31: host check)
                a.tile0 = int(at - before) - a.segment * a.seg_tiles;
                const long long left = end - at;
                a.tile1 = a.seg_tiles - a.tile0 < left ? a.seg_tiles : a.tile0 + int(left);
                a.opens = at == run * blockIdx.x;
                at += a.tile1 - a.tile0;
                return a;
            }
            before = behind;
            ++request;
        }
        a.tokens = 0;
        return a;
    };

    // The copies.  Of a piece, this warp takes the 16 tokens from u * 16, u = first, first + 4, ...: `steps` of them.
    int tokens, first, steps, page_ids, in = 0, at_half = 0;
    const int* table;
    const T *k_head, *v_head;
    // copies half n of the steps: the keys of step n / 2, or its values
    auto fetch = [&](int n) {
        const int step = n >> 1;
        if (step < steps) {
            if ((n & 63) == 0) {                // pages of the steps to come: lane i holds that of step 32 * k + i
                const int s = step + lane;
                page_ids = s < steps ? table[((first + s * kWarpsA) * kUnit) >> p.page_shift] : -1;
            }
            const int page = __shfl_sync(~0u, page_ids, step & 31);
            const int token0 = (first + step * kWarpsA) * kUnit;
            const int slot0 = token0 & ((1 << p.page_shift) - 1);
            const int valid = unsigned(page) < unsigned(p.pages) ? min(kUnit, tokens - token0) : 0;
            const T* const src = (n & 1 ? v_head + (valid ? page : 0) * p.v_page : k_head + (valid ? page : 0) * p.k_page);
            const int64_t slot_stride = n & 1 ? p.v_slot : p.k_slot;
            const uint32_t stage = ring + in * S::kHalf;
            constexpr int kChunks = D / 8;
#pragma unroll
            for (int i = 0; i < kUnit * kChunks / 32; ++i) {
                const int c = i * 32 + lane, row = c / kChunks, col = c % kChunks;
                const uint32_t bytes = row < valid ? 16 : 0;
                const int slot = row < valid ? slot0 + row : 0;
                cp_async16(stage + row * S::kRow + col * 16, src + slot * slot_stride + col * 8, bytes, hint);
            }
        }
        cp_async_commit();
        in = in + 1 == S::kHalves ? 0 : in + 1;
    };
    // queries: row lane / 4 (and + 8), as the first operand of the products with 16 values each
    uint32_t q[D / 16][2 * NT];
    int head0, rows;
    auto begin_piece = [&](const Piece& a) {
        const int kv_head = a.segment / groups, group = a.segment - kv_head * groups;
        tokens = a.tokens;
        first = a.tile0 * kWarpsA + warp;
        const int units = min(a.tile1 * kWarpsA, (tokens + kUnit - 1) / kUnit);
        steps = first < units ? (units - first + kWarpsA - 1) / kWarpsA : 0;
        table = p.block_table + a.request * p.table_stride;
        k_head = static_cast<const T*>(p.k_cache) + kv_head * p.k_head;
        v_head = static_cast<const T*>(p.v_cache) + kv_head * p.v_head;
        in = at_half;                           // (the ring is empty)
#pragma unroll
        for (int n = 0; n < S::kHalves - 1; ++n) fetch(n);
        head0 = kv_head * group_size + group * S::kRows;
        rows = min(S::kRows, group_size - group * S::kRows);
        const uint32_t* row[2];
        bool on[2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int h = lane / 4 + 8 * n;
            on[n] = h < rows;
            row[n] = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + a.request * p.q_request + (head0 + (on[n] ? h : 0)) * p.q_head) + lane % 4;
        }
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                q[k][n] = on[n] ? row[n][k * 8] : 0u;
                q[k][NT + n] = on[n] ? row[n][k * 8 + 4] : 0u;
            }
    };

    Piece piece;
    if constexpr (SHARED) {
        const int mine = int(blockIdx.x) / shares, rank = int(blockIdx.x) - mine * shares;
        piece.request = mine / geo.segments;
        piece.segment = mine - piece.request * geo.segments;
        piece.tokens = geo.tokens(piece.request);
        piece.seg_tiles = (piece.tokens + kTile - 1) / kTile;
        const int each = (piece.seg_tiles + shares - 1) / shares;
        piece.tile0 = min(rank * each, piece.seg_tiles);
        piece.tile1 = min(piece.tile0 + each, piece.seg_tiles);
        piece.opens = true;
    } else {
        piece = next_piece();
    }
    begin_piece(piece);
    while (true) {
        Piece next{};
        if constexpr (!SHARED) next = next_piece();
        // output, turned round: 16 values of a head times 8 heads to a tile
        float o[NT][D / 16][4], m[NT], l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][t][i] = 0.f;
            m[n] = -INFINITY;
            l[n] = 0.f;
        }

        // both products take 8 x 8 blocks of a stage in the same order: tokens 0-7 and 8-15, of each two runs of eight values
        const uint32_t in_stage = ((lane & 7) + ((lane >> 4) & 1) * 8) * S::kRow + ((lane >> 3) & 1) * 16;
        auto next_half = [&](int n) {
            cp_async_wait<S::kHalves - 2>();
            __syncwarp();                       // the half's copies are there, and every lane is done with the one before
            fetch(n + S::kHalves - 1);
            const uint32_t stage = ring + at_half * S::kHalf + in_stage;
            at_half = at_half + 1 == S::kHalves ? 0 : at_half + 1;
            return stage;
        };
        for (int step = 0; step < steps; ++step) {
            // scores of 16 tokens: two products of 8 tokens each, in two chains
            const uint32_t k_at = next_half(2 * step);
            float s[2][2][4];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[c][n][i] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t b0, b1, b2, b3;
                ldmatrix_x4(k_at + k * 32, b0, b1, b2, b3);
                if constexpr (NT == 1) {
                    mma16816<T>(s[k & 1][0], q[k][0], 0u, q[k][1], 0u, b0, b1);
                    mma16816<T>(s[k & 1][1], q[k][0], 0u, q[k][1], 0u, b2, b3);
                } else {
                    mma16816<T>(s[k & 1][0], q[k][0], q[k][1], q[k][2], q[k][3], b0, b1);
                    mma16816<T>(s[k & 1][1], q[k][0], q[k][1], q[k][2], q[k][3], b2, b3);
                }
            }
            const int valid = tokens - (first + step * kWarpsA) * kUnit;
            float alpha[NT];
            uint32_t weight[NT][2][kTerms<T, NT>];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = (s[0][i >> 1][2 * n + (i & 1)] + s[1][i >> 1][2 * n + (i & 1)]) * scale;
                if (valid < kUnit) {
                    const int t = (lane % 4) * 2;
                    if (t >= valid) x[0] = -INFINITY;
                    if (t + 1 >= valid) x[1] = -INFINITY;
                    if (t + 8 >= valid) x[2] = -INFINITY;
                    if (t + 9 >= valid) x[3] = -INFINITY;
                }
                const float top = fmaxf(m[n], quad_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))));
                const float ref = top == -INFINITY ? 0.f : top;       // (nothing but weights of zero so far)
                alpha[n] = exp2f(m[n] - ref);
                m[n] = top;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = exp2f(x[i] - ref);
                l[n] = l[n] * alpha[n] + ((x[0] + x[1]) + (x[2] + x[3]));
                split2<T>(x[0] * kWeightUp<T>, x[1] * kWeightUp<T>, weight[n][0]);
                split2<T>(x[2] * kWeightUp<T>, x[3] * kWeightUp<T>, weight[n][1]);
            }
            bool same = alpha[0] == 1.f;
            if constexpr (NT == 2) same = same && alpha[1] == 1.f;
            if (!__all_sync(~0u, same)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // of the two heads whose values this lane holds
                    const float a0 = __shfl_sync(~0u, alpha[n], (lane % 4) * 8), a1 = __shfl_sync(~0u, alpha[n], (lane % 4) * 8 + 4);
#pragma unroll
                    for (int t = 0; t < D / 16; ++t) {
                        o[n][t][0] *= a0;
                        o[n][t][1] *= a1;
                        o[n][t][2] *= a0;
                        o[n][t][3] *= a1;
                    }
                }
            }
            const uint32_t v_at = next_half(2 * step + 1);
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                uint32_t a0, a1, a2, a3;
                ldmatrix_x4_trans(v_at + t * 32, a0, a1, a2, a3);
#pragma unroll
                for (int i = 0; i < kTerms<T, NT>; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816<T>(o[n][t], a0, a1, a2, a3, weight[n][0][i], weight[n][1][i]);
            }
        }
        const int out_head = head0, out_rows = rows;
        if constexpr (S::kApart) {
            if (next.tokens) begin_piece(next);
        } else {
            cp_async_wait<0>();
            __syncthreads();                    // the rings are free
        }

        // the warps' results: maxima and sums, outputs
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float sum = quad_sum(l[n]);
            if (lane % 4 == 0) join_ml[warp * S::kRows + lane / 4 + 8 * n] = make_float2(m[n], sum);
            float* const at_head = join + (warp * S::kRows + (lane % 4) * 2 + 8 * n) * S::kJoinRow + lane / 4;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                at_head[t * 16] = o[n][t][0];
                at_head[t * 16 + S::kJoinRow] = o[n][t][1];
                at_head[t * 16 + 8] = o[n][t][2];
                at_head[t * 16 + 8 + S::kJoinRow] = o[n][t][3];
            }
        }
        __syncthreads();
        // (more than one CTA: the rest is joined by join_kernel)
        const bool whole = piece.tile0 == 0 && piece.tile1 == piece.seg_tiles;
        float* const part = static_cast<float*>(p.workspace) + (int64_t(blockIdx.x) * 2 + (piece.opens ? 0 : 1)) * S::kPart;
        for (int i = threadIdx.x; i < out_rows * (D / 2); i += kThreadsA) {
            const int row = i / (D / 2), c = (i % (D / 2)) * 2;
            float2 ml[kWarpsA];
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarpsA; ++w) {
                ml[w] = join_ml[w * S::kRows + row];
                top = fmaxf(top, ml[w].x);
            }
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            float2 v = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarpsA; ++w) {
                const float f = exp2f(ml[w].x - ref);
                const float2 x = *reinterpret_cast<const float2*>(join + (w * S::kRows + row) * S::kJoinRow + c);
                sum += f * ml[w].y;
                v.x += f * x.x;
                v.y += f * x.y;
            }
            if constexpr (SHARED) {             // kept where warp 0's was, for the cluster
                *reinterpret_cast<float2*>(join + row * S::kJoinRow + c) = v;
                if (c == 0) share_ml[row] = make_float2(top, sum);
            } else if (whole) {
                const float inv = 1.f / kWeightUp<T> / sum;
                *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (int64_t(piece.request) * p.heads + out_head + row) * D + c) = pack2<T>(v.x * inv, v.y * inv);
            } else {
                *reinterpret_cast<float2*>(part + row * D + c) = v;
                if (c == 0) *reinterpret_cast<float2*>(part + S::kRows * D + row * 2) = make_float2(top, sum);
            }
        }
        if constexpr (SHARED) {
            __syncthreads();
            cluster_arrive_release();
            cluster_wait_acquire();             // every share's result is in its CTA's shared memory
            const int rank = int(cluster_ctarank());
            for (int i = rank * kThreadsA + int(threadIdx.x); i < out_rows * (D / 2); i += shares * kThreadsA) {
                const int row = i / (D / 2), c = (i % (D / 2)) * 2;
                const uint32_t at_v = smem_u32(join + row * S::kJoinRow + c), at_ml = smem_u32(&share_ml[row]);
                float2 ml[kMostShares], x[kMostShares];
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kMostShares; ++w) {
                    ml[w] = w < shares ? ld_cluster_f2(mapa(at_ml, w)) : make_float2(-INFINITY, 0.f);
                    x[w] = w < shares ? ld_cluster_f2(mapa(at_v, w)) : make_float2(0.f, 0.f);
                    top = fmaxf(top, ml[w].x);
                }
                const float ref = top == -INFINITY ? 0.f : top;
                float sum = 0.f;
                float2 v = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kMostShares; ++w) {
                    const float f = exp2f(ml[w].x - ref);
                    sum += f * ml[w].y;
                    v.x += f * x[w].x;
                    v.y += f * x[w].y;
                }
                const float inv = piece.tokens ? 1.f / kWeightUp<T> / sum : 0.f;        // (no tokens: zeros)
                *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (int64_t(piece.request) * p.heads + out_head + row) * D + c) = pack2<T>(v.x * inv, v.y * inv);
            }
            __syncwarp();
            cluster_arrive_release();
            cluster_wait_acquire();             // nobody reads this CTA's shared memory any more
        }
        if (!next.tokens) break;
        __syncthreads();                        // the join's memory is written again
        if constexpr (!S::kApart) begin_piece(next);
        piece = next;
    }
    cp_async_wait<0>();
}

// Where a head's partial results are: `parts` of them, in the slots of runs `run`, run + 1, ...
struct Pieces {
    int parts, run, first_slot, request, head, row;
};

// Joins the runs over which segments were cut: `per_cta` (1, or a multiple of 8 up to 64) query heads to a CTA.  It is launched while
// the first kernel still runs and finds its place in the work meanwhile.  A warp joins a head of few parts by itself, all warps of the
// CTA one of many; maxima come first, so that the loads of the parts do not wait for one another.  Sums run in the order of the
// tokens.  (Behind the first kernel it takes 3 us, 12 for 19200 heads; with eight heads to a CTA those take 24.  A CTA to each run, for
// the segment that is cut at its end: 7 us more for 2400 heads.)
template <typename T, int D, int NT, bool MANY>
__global__ void __launch_bounds__(kThreadsJ, MANY ? 4 : 1) join_kernel(const __grid_constant__ PagedAttention p, int groups, const Cut cut, int per_cta) {
    using S = Shape<D, NT>;
    constexpr int kColumns = (D / 4 + 31) / 32;          // of four values, per lane
    constexpr int kBatch = (MANY ? 8 : 16) / kColumns;   // loads in flight
    constexpr int kFew = 16;
    __shared__ long long scratch[kWarpsJ], before[kMostHeads];
    __shared__ Pieces found[kWarpsJ];
    __shared__ float2 ml[kMostParts];
    __shared__ float highest[kWarpsJ], sums[kWarpsJ];
    __shared__ float4 share[kWarpsJ][D / 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group_size = p.heads / p.kv_heads, first_head = int(blockIdx.x) * per_cta;
    const int last_head = min(p.requests * p.heads - first_head, per_cta) + first_head;
    const Geometry geo{p.lengths, p.requests, p.kv_heads * groups, (long long)p.columns << p.page_shift};
    const int first_request = first_head / p.heads;
    long long total = 0;
    for (int r0 = 0; r0 < p.requests; r0 += kThreadsJ * kEach) {
        const int r = r0 + int(threadIdx.x) * kEach;
        int tiles[kEach];
        long long here, at = total + scan_tiles<kWarpsJ>(geo.some(r, tiles), scratch, &here);
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (r + k >= first_request && r + k < first_request + per_cta) before[r + k - first_request] = at;
            at += tiles[k];
        }
        total += here;
    }
    __syncthreads();
    const long long run = cut.run(total);
    auto pieces_of = [&](int h) {
        Pieces a{};
        const int request = h / p.heads, head = h - request * p.heads;
        const int kv_head = head / group_size, in_group = head - kv_head * group_size;
        const int segment = kv_head * groups + in_group / S::kRows;
        const int seg_tiles = (geo.tokens(request) + kTile - 1) / kTile;
        if (seg_tiles) {
            const long long begin = before[request - first_request] + (long long)segment * seg_tiles;
            const int first = int(begin / run), last = int((begin + seg_tiles - 1) / run);
            // the segment opens its first run unless it begins inside it
            a = {last - first + 1, first, begin <= run * first ? 0 : 1, request, head, in_group % S::kRows};
        }
        return a;
    };
    // (every CTA waits for the first kernel, so that this one ends after it, and what follows on the stream after both)
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const float* const workspace = static_cast<const float*>(p.workspace);
    auto part_of = [&](const Pieces& a, int i) { return workspace + (int64_t(a.run + i) * 2 + (i == 0 ? a.first_slot : 0)) * S::kPart; };
    auto ml_of = [&](const Pieces& a, int i) { return *reinterpret_cast<const float2*>(part_of(a, i) + S::kRows * D + a.row * 2); };
    // this lane's columns of a part's row
    auto load = [&](const Pieces& a, int i, bool real, float4 (&x)[kColumns]) {
#pragma unroll
        for (int k = 0; k < kColumns; ++k) {
            const int c = k * 32 + lane;
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (real && c < D / 4) x[k] = *reinterpret_cast<const float4*>(part_of(a, i) + a.row * D + c * 4);
        }
    };
    auto add = [](float4 (&v)[kColumns], float f, const float4 (&x)[kColumns]) {
#pragma unroll
        for (int k = 0; k < kColumns; ++k) {
            v[k].x += f * x[k].x;
            v[k].y += f * x[k].y;
            v[k].z += f * x[k].z;
            v[k].w += f * x[k].w;
        }
    };
    auto write = [&](const Pieces& a, int c, float4 v, float inv) {
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (int64_t(a.request) * p.heads + a.head) * D + c * 4) =
            make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
    };
    auto warp_max = [](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
        return x;
    };
    auto warp_sum = [](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
        return x;
    };

    for (int h0 = first_head; h0 < last_head; h0 += kWarpsJ) {
        Pieces mine{};
        if (h0 + warp < last_head) mine = pieces_of(h0 + warp);
        if (lane == 0) found[warp] = mine;
        if (mine.parts > 1 && mine.parts <= kFew) {
            const float2 m = lane < mine.parts ? ml_of(mine, lane) : make_float2(-INFINITY, 0.f);
            const float top = warp_max(m.x), f = exp2f(m.x - (top == -INFINITY ? 0.f : top)), sum = warp_sum(f * m.y);
            float4 v[kColumns] = {};
            for (int i0 = 0; i0 < mine.parts; i0 += kBatch) {
                float4 x[kBatch][kColumns];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) load(mine, i0 + i, i0 + i < mine.parts, x[i]);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) add(v, __shfl_sync(~0u, f, (i0 + i) & 31), x[i]);      // (0 behind the last part)
            }
#pragma unroll
            for (int k = 0; k < kColumns; ++k)
                if (k * 32 + lane < D / 4) write(mine, k * 32 + lane, v[k], 1.f / kWeightUp<T> / sum);
        }
        if (!__syncthreads_or(mine.parts > kFew)) continue;
        for (int w = 0; w < kWarpsJ; ++w) {
            const Pieces a = found[w];
            if (a.parts <= kFew) continue;
            float top = -INFINITY;
            for (int i = threadIdx.x; i < a.parts; i += kThreadsJ) {
                ml[i] = ml_of(a, i);
                top = fmaxf(top, ml[i].x);
            }
            top = warp_max(top);
            if (lane == 0) highest[warp] = top;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kWarpsJ; ++k) top = fmaxf(top, highest[k]);
            const float ref = top == -INFINITY ? 0.f : top;
            const int per = (a.parts + kWarpsJ - 1) / kWarpsJ, lo = warp * per, hi = min(a.parts, lo + per);
            float4 v[kColumns] = {};
            float sum = 0.f;
            for (int i0 = lo; i0 < hi; i0 += kBatch) {
                float4 x[kBatch][kColumns];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) load(a, i0 + i, i0 + i < hi, x[i]);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const float2 m = i0 + i < hi ? ml[i0 + i] : make_float2(-INFINITY, 0.f);
                    const float f = exp2f(m.x - ref);
                    sum += f * m.y;
                    add(v, f, x[i]);
                }
            }
#pragma unroll
            for (int k = 0; k < kColumns; ++k)
                if (k * 32 + lane < D / 4) share[warp][k * 32 + lane] = v[k];
            if (lane == 0) sums[warp] = sum;
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int k = 0; k < kWarpsJ; ++k) sum += sums[k];
            const float inv = 1.f / kWeightUp<T> / sum;
            for (int c = threadIdx.x; c < D / 4; c += kThreadsJ) {
                float4 x = share[0][c];
#pragma unroll
                for (int k = 1; k < kWarpsJ; ++k) {
                    const float4 y = share[k][c];
                    x.x += y.x;
                    x.y += y.y;
                    x.z += y.z;
                    x.w += y.w;
                }
                write(a, c, x, inv);
            }
            __syncthreads();                                 // the next head's turn
        }
        __syncthreads();                                     // everyone has read what was found
    }
}

template <typename T, int D, int NT>
cudaError_t launch(const PagedAttention& a, int num_sms, cudaStream_t stream) {
    using S = Shape<D, NT>;
    const int group_size = a.heads / a.kv_heads, groups = (group_size + S::kRows - 1) / S::kRows;
    const long long segments = (long long)a.requests * a.kv_heads * groups, resident = S::kCtasPerSm * min(num_sms, kMostSms);
    // what the table could hold, in tiles of a segment
    const long long tiles = (((long long)a.columns << a.page_shift) + kTile - 1) / kTile;
    int shares = 1;
    while (shares < kMostShares && shares < tiles && segments * shares * 2 <= resident) shares *= 2;
    if (tiles <= kShort * shares && segments * shares <= 0x7fffffff) {
        auto kern = paged_attention_kernel<T, D, NT, true>;
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e != cudaSuccess) return e;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim = {unsigned(shares), 1, 1};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(segments * shares));
        cfg.blockDim = dim3(kThreadsA);
        cfg.dynamicSmemBytes = S::kSmem;
        cfg.stream = stream;
        cfg.attrs = &cluster;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kern, a, groups, Cut{}, shares);
    }
    auto kern = paged_attention_kernel<T, D, NT, false>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    // no more CTAs than the table could hold tiles
    const long long most = segments * tiles < 1 ? 1 : segments * tiles;
    const Cut cut{int(most < resident ? most : resident), kWaves, least_run(D)};
    const int ctas = int(most < (long long)cut.resident * kWaves ? most : (long long)cut.resident * kWaves);
    kern<<<ctas, kThreadsA, S::kSmem, stream>>>(a, groups, cut, 1);
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    // a head to a CTA while that is a few CTAs for each SM at most
    // (and as many as keep it so, beyond)
    const long long heads = (long long)a.requests * a.heads, most_ctas = 4 * num_sms;
    long long per = heads <= most_ctas ? 1 : (heads + most_ctas - 1) / most_ctas;
    if (per > 1) per = (per + kWarpsJ - 1) / kWarpsJ * kWarpsJ;
    const int per_cta = int(per < kMostHeads ? per : kMostHeads);
    cfg.gridDim = dim3(unsigned((heads + per_cta - 1) / per_cta));
    cfg.blockDim = dim3(kThreadsJ);
    cfg.stream = stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, per_cta > 1 ? join_kernel<T, D, NT, true> : join_kernel<T, D, NT, false>, a, groups, cut, per_cta);
}

template <typename T, int D>
cudaError_t launch_d(const PagedAttention& a, int num_sms, cudaStream_t stream) {
    return a.heads / a.kv_heads <= 8 ? launch<T, D, 1>(a, num_sms, stream) : launch<T, D, 2>(a, num_sms, stream);
}

template <typename T>
cudaError_t launch_t(const PagedAttention& a, int num_sms, cudaStream_t stream) {
    switch (a.dim) {
        case 64: return launch_d<T, 64>(a, num_sms, stream);
        case 96: return launch_d<T, 96>(a, num_sms, stream);
        case 128: return launch_d<T, 128>(a, num_sms, stream);
        case 256: return launch_d<T, 256>(a, num_sms, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

bool paged_attention_supported(int heads, int kv_heads, int dim) {
    return kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && (dim == 64 || dim == 96 || dim == 128 || dim == 256);
}

size_t paged_attention_workspace_bytes(int heads, int kv_heads, int dim, int num_sms) {
    const int rows = heads / kv_heads <= 8 ? 8 : 16;
    return size_t(ctas_per_sm(dim, heads / kv_heads <= 8 ? 1 : 2)) * (num_sms < kMostSms ? num_sms : kMostSms) * kWaves * 2 * rows * (dim + 2) * sizeof(float);
}

cudaError_t paged_attention(const PagedAttention& a, int num_sms, cudaStream_t stream) {
    return a.f16 ? launch_t<__half>(a, num_sms, stream) : launch_t<__nv_bfloat16>(a, num_sms, stream);
}

}  // namespace dlr
