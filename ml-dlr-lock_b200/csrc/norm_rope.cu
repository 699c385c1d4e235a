// RMS norm of every query and key head with the rotation by position in the same pass, its gradient, and the form that puts
// keys and values straight into a paged cache.
//
//   n = x * rsqrt(mean(x^2) + eps) * w             (left out where there is no weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)       over the pairs of the first 2 * half values; the rest passes through
//
// Pairs are (i, i + half), or (2i, 2i + 1) where the layout is interleaved.  Backward, with g the incoming gradient turned
// back by the same angle, u = x * rstd:   dx = rstd * (g w - u * mean(g w u)),   dw = sum of g u over tokens and heads.
//
// Bound by memory: every value is read once and written once.  dim / 16 lanes share a head and each holds two runs of eight values
// that are each other's partners (runs l and l + half / 8, or neighbouring ones), so that the rotation needs no exchange between
// lanes, and a lane needs 8 cosines and 8 sines instead of 16 of each.  A warp takes several heads of one token, which share
// those.  Everything between the load and the store is fp32, rounded once.
#include "norm_rope.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace dlr {

namespace {

constexpr int kThreadsN = 128;
constexpr int kWarpsN = kThreadsN / 32;

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t v);
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

template <typename T>
__device__ __forceinline__ uint32_t from_floats(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t from_floats<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t from_floats<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// two fp32 values
struct Pair {
    float x, y;
};
__device__ __forceinline__ Pair pair(float lo, float hi) { return {lo, hi}; }
__device__ __forceinline__ float2 floats(Pair p) { return make_float2(p.x, p.y); }
__device__ __forceinline__ Pair swapped(Pair p) { return {p.y, p.x}; }
__device__ __forceinline__ Pair mul(Pair a, Pair b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) { return {fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)}; }

// A lane's run of RUN neighbouring values of a head, as it lies in memory and as fp32 pairs.
template <int RUN>
struct Raw;
template <>
struct Raw<8> {
    using type = uint4;
};
template <>
struct Raw<4> {
    using type = uint2;
};

template <typename T, int RUN>
__device__ __forceinline__ void unpack(const typename Raw<RUN>::type& raw, Pair (&v)[RUN / 2]) {
    const uint32_t* const w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < RUN / 2; ++i) {
        const float2 f = to_float2<T>(w[i]);
        v[i] = pair(f.x, f.y);
    }
}
template <typename T, int RUN>
__device__ __forceinline__ typename Raw<RUN>::type pack(const Pair (&v)[RUN / 2]) {
    typename Raw<RUN>::type raw;
    uint32_t* const w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < RUN / 2; ++i) {
        const float2 f = floats(v[i]);
        w[i] = from_floats<T>(f.x, f.y);
    }
    return raw;
}

// the two runs that lane l of a head holds, as indexes of values
struct Runs {
    int a, b;
    bool turned;
};

template <int RUN, bool INTERLEAVED>
__device__ __forceinline__ Runs runs_of(int l, int half) {
    Runs r;
    r.turned = l < half / RUN;
    if (INTERLEAVED || !r.turned) {
        r.a = 2 * RUN * l;
        r.b = r.a + RUN;
    } else {
        r.a = RUN * l;
        r.b = r.a + half;
    }
    return r;
}

// What a value and its partner contribute to a turned value: x -> own * x + other * partner, for both runs.  In the half
// layout the partner is the value at the same place of the other run, in the interleaved one the pair's other value.
// SIGN = 1: by the angle; -1: back.  Where a lane's values pass through, own is 1 and other is not used.
template <int RUN, bool INTERLEAVED, int SIGN>
__device__ __forceinline__ void coefficients(const float* c, const float* s, bool turned, Pair (&own)[RUN], Pair (&other)[RUN]) {
    if (!turned) {
#pragma unroll
        for (int j = 0; j < RUN; ++j) {
            own[j] = pair(1.f, 1.f);
            other[j] = {};
        }
    } else if constexpr (INTERLEAVED) {                  // cosine j belongs to the pair (2j, 2j + 1) of the two runs in a row
#pragma unroll
        for (int j = 0; j < RUN; ++j) {
            own[j] = pair(c[j], c[j]);
            other[j] = pair(-SIGN * s[j], SIGN * s[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < RUN / 2; ++i) {
            own[i] = own[RUN / 2 + i] = pair(c[2 * i], c[2 * i + 1]);
            other[i] = pair(-SIGN * s[2 * i], -SIGN * s[2 * i + 1]);
            other[RUN / 2 + i] = pair(SIGN * s[2 * i], SIGN * s[2 * i + 1]);
        }
    }
}

// partner of pair j of the two runs v[0 .. RUN)
template <int RUN, bool INTERLEAVED>
__device__ __forceinline__ Pair partner(const Pair (&v)[RUN], int j) {
    return INTERLEAVED ? swapped(v[j]) : v[j < RUN / 2 ? j + RUN / 2 : j - RUN / 2];
}

template <int RUN>
__device__ __forceinline__ void load_floats(const float* p, Pair (&v)[RUN / 2]) {
#pragma unroll
    for (int i = 0; i < RUN / 4; ++i) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p) + i);
        v[2 * i] = pair(x.x, x.y);
        v[2 * i + 1] = pair(x.z, x.w);
    }
}

// a lane's values of a weight (of one where there is none)
template <typename T, int RUN>
__device__ __forceinline__ void load_weight(const void* w, bool f32, bool on, const Runs& run, Pair (&v)[RUN]) {
#pragma unroll
    for (int i = 0; i < RUN; ++i) v[i] = pair(1.f, 1.f);
    if (!w || !on) return;
    Pair a[RUN / 2], b[RUN / 2];
    if (f32) {
        load_floats<RUN>(static_cast<const float*>(w) + run.a, a);
        load_floats<RUN>(static_cast<const float*>(w) + run.b, b);
    } else {
        using R = typename Raw<RUN>::type;
        unpack<T, RUN>(__ldg(reinterpret_cast<const R*>(static_cast<const T*>(w) + run.a)), a);
        unpack<T, RUN>(__ldg(reinterpret_cast<const R*>(static_cast<const T*>(w) + run.b)), b);
    }
#pragma unroll
    for (int i = 0; i < RUN / 2; ++i) {
        v[i] = a[i];
        v[RUN / 2 + i] = b[i];
    }
}

template <typename T, int RUN>
__device__ __forceinline__ void unpack_both(const typename Raw<RUN>::type& ra, const typename Raw<RUN>::type& rb, bool real, Pair (&v)[RUN]) {
    Pair a[RUN / 2] = {}, b[RUN / 2] = {};
    if (real) {
        unpack<T, RUN>(ra, a);
        unpack<T, RUN>(rb, b);
    }
#pragma unroll
    for (int i = 0; i < RUN / 2; ++i) {
        v[i] = a[i];
        v[RUN / 2 + i] = b[i];
    }
}

template <typename T, int RUN>
__device__ __forceinline__ void pack_both(const Pair (&v)[RUN], typename Raw<RUN>::type& ra, typename Raw<RUN>::type& rb) {
    Pair a[RUN / 2], b[RUN / 2];
#pragma unroll
    for (int i = 0; i < RUN / 2; ++i) {
        a[i] = v[i];
        b[i] = v[RUN / 2 + i];
    }
    ra = pack<T, RUN>(a);
    rb = pack<T, RUN>(b);
}

__device__ __forceinline__ float sum_of(Pair p) {
    const float2 f = floats(p);
    return f.x + f.y;
}

__device__ __forceinline__ int64_t position_of(const void* positions, bool is64, int64_t t) {
    return is64 ? static_cast<const long long*>(positions)[t] : (long long)static_cast<const int*>(positions)[t];
}

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// ---- the lanes' queues --------------------------------------------------------------------------------------------------
// A warp walks over units of (token, group of up to U * 32 / LPH heads).  Its lanes copy what the next unit needs into a queue in
// shared memory (cp.async) while they work on this one, so that loads are in flight all the time without registers for them.  What
// the heads of a unit share (angles times weights) is formed once.  5001 tokens, 64 + 8 heads of 128 with values: 39 us, of 31.6 at
// copy bandwidth (a plain elementwise pass over as many bytes takes 33, and so does this loop without the arithmetic 39: what is
// left is its pattern of loads and stores); 8192 tokens, 32 + 8 heads: 31 us of 25.6, backward 50 of 38.4.  With loads into
// registers, unit after unit: 46, 38 and 82.  Arithmetic on register pairs written as such (f32x2) was slower: 41, 33 and 50.
__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(shared_address(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One unit's share of a warp's queue: V runs of RUN values per lane, and for the lanes of one head its cosines and sines (the
// heads side by side share them).
template <int RUN, int LPH, int V>
struct Stage {
    typename Raw<RUN>::type runs[V][32];
    float4 cos[RUN / 4][LPH], sin[RUN / 4][LPH];
    int slot[4];
};

constexpr int kStagesN = 2;
// Heads one behind the other in a unit, and blocks of an SM.  Measured for 5001 tokens, 64 + 8 heads of 128 with values, and 8192
// tokens, 32 + 8 heads (us): 39 / 31 with units of 4 and 4 or 5 blocks, 54 / 44 with 6 (registers spill), 39 / 32 with twice as
// many blocks as are resident; 10 and more us longer with units of 2 or 8, or a queue of three units (fewer warps fit).  Backward:
// 50 with units of 2 and 3 or 4 blocks, 67 with 5, 56 with units of 1, 67 with units of 4.
constexpr int kForwardUnit = 4, kForwardBlocksPerSm = 5, kBackwardUnit = 2, kBackwardBlocks = 3;

// The units of a warp: the `stride`-th next one each time, without a division.
struct Walk {
    int64_t token;
    int group, groups, token_step, group_step;

    __device__ __forceinline__ Walk(int64_t first, int64_t stride, int groups) : groups(groups) {
        token = first / groups;
        group = int(first - token * groups);
        token_step = int(stride / groups);
        group_step = int(stride - int64_t(token_step) * groups);
    }
    __device__ __forceinline__ void next() {
        token += token_step;
        group += group_step;
        if (group >= groups) {
            group -= groups;
            ++token;
        }
    }
};

// Cosines and sines for a unit to come: each lane copies those of its pairs, for the lanes like it in the other heads too.
template <int RUN, int LPH, int V>
__device__ __forceinline__ void fetch_angles(Stage<RUN, LPH, V>& st, const float* cos, const float* sin, int half, int rows, int64_t position,
                                             bool mine, int l) {
    if (mine && position >= 0 && position < rows) {
        const int64_t at = position * half + RUN * l;
#pragma unroll
        for (int i = 0; i < RUN / 4; ++i) {
            copy_async<16>(&st.cos[i][l], cos + at + 4 * i);
            copy_async<16>(&st.sin[i][l], sin + at + 4 * i);
        }
    }
}

// A position outside the tables makes the row NaN.
template <int RUN, bool INTERLEAVED, int SIGN, int LPH, int V>
__device__ __forceinline__ void take_angles(const Stage<RUN, LPH, V>& st, bool known, bool turned, int l, Pair (&own)[RUN], Pair (&other)[RUN]) {
    float c[RUN], s[RUN];
    if (turned) {
#pragma unroll
        for (int i = 0; i < RUN / 4; ++i) {
            const float4 x = st.cos[i][l], y = st.sin[i][l];
            c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
            s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
        }
    }
    coefficients<RUN, INTERLEAVED, SIGN>(c, s, turned, own, other);
    if (!known) {
        const Pair nan = pair(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
#pragma unroll
        for (int j = 0; j < RUN; ++j) own[j] = nan;
    }
}

// Groups are those of the queries, then the keys, then the values.
template <typename T, int RUN, int LPH, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreadsN, kForwardBlocksPerSm) norm_rope_kernel(const __grid_constant__ NormRope p, int q_groups, int k_groups, int groups) {
    constexpr int kSide = 32 / LPH;                      // heads side by side in a warp
    extern __shared__ __align__(16) uint8_t memory[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPH, sub = lane / LPH;
    using R = typename Raw<RUN>::type;
    using Unit = Stage<RUN, LPH, 2 * U>;
    Unit* const queue = reinterpret_cast<Unit*>(memory) + warp * kStagesN;
    const Runs run = runs_of<RUN, INTERLEAVED>(l, p.half);
    const bool lane_on = 2 * RUN * l < p.dim, turned = run.turned && lane_on;
    const int64_t first_unit = int64_t(blockIdx.x) * kWarpsN + warp, stride = int64_t(gridDim.x) * kWarpsN;
    const int gap = run.b - run.a;
    Walk ahead(first_unit, stride, groups), now = ahead;
    const float inv = 1.0f / float(p.dim);

    auto kind_of = [&](int group) { return group < q_groups ? 0 : group < q_groups + k_groups ? 1 : 2; };
    auto group_in = [&](int group, int kind) { return group - (kind == 0 ? 0 : kind == 1 ? q_groups : q_groups + k_groups); };
    int stage_in = 0, stage_out = 0;
    unsigned known_in = 0;                               // whether the position of the unit in a stage is in the tables, by stage
    auto fetch = [&](int64_t position) {
        if (ahead.token < p.tokens) {
            Unit& st = queue[stage_in];
            const int kind = kind_of(ahead.group), first = group_in(ahead.group, kind) * (U * kSide) + sub;
            const Heads& in = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
            const int left = (kind == 0 ? p.q_heads : p.k_heads) - first;
            const T* x = static_cast<const T*>(in.data) + ahead.token * in.token + first * in.head + run.a;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (lane_on && u * kSide < left) {
                    copy_async<2 * RUN>(&st.runs[2 * u][lane], x);
                    copy_async<2 * RUN>(&st.runs[2 * u + 1][lane], x + gap);
                }
                x += kSide * in.head;
            }
            fetch_angles(st, p.cos, p.sin, p.half, p.table_rows, position, turned && kind != 2 && sub == 0, l);
            if (p.slots && kind != 0 && lane == 0) copy_async<4>(st.slot, p.slots + ahead.token);
        }
        const bool known = position >= 0 && position < p.table_rows;
        known_in = (known_in & ~(1u << stage_in)) | (unsigned(known) << stage_in);
        copies_commit();
        ahead.next();
        stage_in = stage_in + 1 == kStagesN ? 0 : stage_in + 1;
    };
    // the position of the unit that is fetched next
    auto position_ahead = [&]() { return ahead.token < p.tokens ? position_of(p.positions, p.positions_64, ahead.token) : 0; };
    for (int i = 0; i < kStagesN - 1; ++i) fetch(position_ahead());
    int64_t position = position_ahead();

    for (; now.token < p.tokens; now.next()) {
        copies_wait<kStagesN - 2>();
        __syncwarp();                                    // every lane's copies are there, and all are done with the unit before
        const bool known = (known_in >> stage_out) & 1u;
        fetch(position);
        position = position_ahead();
        Unit& st = queue[stage_out];
        stage_out = stage_out + 1 == kStagesN ? 0 : stage_out + 1;
        const int kind = kind_of(now.group), base = group_in(now.group, kind) * (U * kSide), first = base + sub;
        const int heads = kind == 0 ? p.q_heads : p.k_heads;
        const int64_t token = now.token;
        // where the unit's heads go, `step` values apart: to q_out or k_out, or to the token's slot of the cache; keys may go to both
        T* to = kind == 0 ? static_cast<T*>(p.q_out) + (token * p.q_heads + first) * p.dim + run.a : nullptr;
        T* also = nullptr;
        int64_t step = kSide * p.dim;
        if (kind != 0) {
            if (kind == 1 && p.k_out) also = static_cast<T*>(p.k_out) + (token * p.k_heads + first) * p.dim + run.a;
            const int64_t slot = p.slots ? st.slot[0] : -1;
            if (slot >= 0 && slot < p.n_slots) {             // (a row without a place in the cache otherwise)
                const int64_t page = slot >> p.page_shift, at = slot & ((1 << p.page_shift) - 1);
                to = (kind == 1 ? static_cast<T*>(p.k_cache) + page * p.k_page + at * p.k_slot + first * p.k_head
                                : static_cast<T*>(p.v_cache) + page * p.v_page + at * p.v_slot + first * p.v_head) + run.a;
                step = kSide * (kind == 1 ? p.k_head : p.v_head);
            } else {
                to = also;
                also = nullptr;
            }
            if (!to) continue;
        }
        // (of the u-th heads side by side, in turn)
        auto store = [&](bool real, const R& a, const R& b) {
            if (real) {
                *reinterpret_cast<R*>(to) = a;
                *reinterpret_cast<R*>(to + gap) = b;
            }
            to += step;
            if (also) {
                if (real) {
                    *reinterpret_cast<R*>(also) = a;
                    *reinterpret_cast<R*>(also + gap) = b;
                }
                also += kSide * p.dim;
            }
        };
        if (kind == 2) {
#pragma unroll
            for (int u = 0; u < U; ++u) store(lane_on && first + u * kSide < heads, st.runs[2 * u][lane], st.runs[2 * u + 1][lane]);
        } else {
            // the weights go into the coefficients, which all heads of the unit share; what is left to each is its rstd
            Pair own[RUN], other[RUN], w[RUN];
            const void* const weight = kind == 0 ? p.q_weight : p.k_weight;
            take_angles<RUN, INTERLEAVED, 1>(st, known, turned, l, own, other);
            if (weight) {
                load_weight<T, RUN>(weight, p.weights_f32, lane_on, run, w);
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    own[j] = mul(own[j], w[j]);
                    other[j] = mul(other[j], partner<RUN, INTERLEAVED>(w, j));
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (base + u * kSide >= heads) break;
                const bool real = lane_on && first + u * kSide < heads;
                Pair v[RUN], y[RUN];
                unpack_both<T, RUN>(st.runs[2 * u][lane], st.runs[2 * u + 1][lane], real, v);
                Pair scale{};
                if (weight) {
                    Pair ss{};
#pragma unroll
                    for (int j = 0; j < RUN; ++j) ss = fma(v[j], v[j], ss);
                    const float rstd = rsqrtf(head_sum<LPH>(sum_of(ss)) * inv + p.eps);
                    scale = pair(rstd, rstd);
                }
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    y[j] = mul(own[j], v[j]);
                    if (turned) y[j] = fma(other[j], partner<RUN, INTERLEAVED>(v, j), y[j]);
                    if (weight) y[j] = mul(y[j], scale);
                }
                R a, b;
                pack_both<T, RUN>(y, a, b);
                store(real, a, b);
            }
        }
    }
    copies_wait<0>();
}

// Blocks of the first q_blocks take query heads, the others key heads; a warp keeps its share of the weight's gradient in
// registers.  Shares are added up in a fixed order: shuffles, the block's warps, and (weight_gradient_kernel) the blocks, so
// that results repeat bit for bit.
template <typename T, int RUN, int LPH, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreadsN, kBackwardBlocks) norm_rope_backward_kernel(const __grid_constant__ NormRopeBackward p, int q_blocks) {
    constexpr int kSide = 32 / LPH;
    extern __shared__ __align__(16) uint8_t memory[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPH, sub = lane / LPH;
    using R = typename Raw<RUN>::type;
    using Unit = Stage<RUN, LPH, 4 * U>;
    Unit* const queue = reinterpret_cast<Unit*>(memory) + warp * kStagesN;
    asm volatile("griddepcontrol.launch_dependents;");
    const bool keys = int(blockIdx.x) >= q_blocks;
    const int block = keys ? int(blockIdx.x) - q_blocks : int(blockIdx.x), blocks = keys ? int(gridDim.x) - q_blocks : q_blocks;
    const Heads& in = keys ? p.k : p.q;
    const Heads& grad = keys ? p.k_grad : p.q_grad;
    const void* const weight = keys ? p.k_weight : p.q_weight;
    T* const dx = static_cast<T*>(keys ? p.dk : p.dq);
    const int heads = keys ? p.k_heads : p.q_heads, groups = (heads + U * kSide - 1) / (U * kSide);
    const Runs run = runs_of<RUN, INTERLEAVED>(l, p.half);
    const bool lane_on = 2 * RUN * l < p.dim, turned = run.turned && lane_on;
    Pair w[RUN], dw[RUN] = {};
    load_weight<T, RUN>(weight, p.weights_f32, lane_on, run, w);
    const float inv = 1.0f / float(p.dim);
    Walk ahead(int64_t(block) * kWarpsN + warp, int64_t(blocks) * kWarpsN, groups), now = ahead;

    int stage_in = 0, stage_out = 0;
    unsigned known_in = 0;                               // whether the position of the unit in a stage is in the tables, by stage
    auto fetch = [&](int64_t position) {
        if (ahead.token < p.tokens) {
            Unit& st = queue[stage_in];
            const int first = ahead.group * (U * kSide) + sub;
            const T* g = static_cast<const T*>(grad.data) + ahead.token * grad.token + first * grad.head;
            const T* x = static_cast<const T*>(in.data) + ahead.token * in.token + first * in.head;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (lane_on && first + u * kSide < heads) {
                    copy_async<2 * RUN>(&st.runs[4 * u][lane], g + run.a);
                    copy_async<2 * RUN>(&st.runs[4 * u + 1][lane], g + run.b);
                    if (weight) {
                        copy_async<2 * RUN>(&st.runs[4 * u + 2][lane], x + run.a);
                        copy_async<2 * RUN>(&st.runs[4 * u + 3][lane], x + run.b);
                    }
                }
                g += kSide * grad.head;
                x += kSide * in.head;
            }
            fetch_angles(st, p.cos, p.sin, p.half, p.table_rows, position, turned && sub == 0, l);
        }
        const bool known = position >= 0 && position < p.table_rows;
        known_in = (known_in & ~(1u << stage_in)) | (unsigned(known) << stage_in);
        copies_commit();
        ahead.next();
        stage_in = stage_in + 1 == kStagesN ? 0 : stage_in + 1;
    };
    auto position_ahead = [&]() { return ahead.token < p.tokens ? position_of(p.positions, p.positions_64, ahead.token) : 0; };
    for (int i = 0; i < kStagesN - 1; ++i) fetch(position_ahead());
    int64_t position = position_ahead();

    for (; now.token < p.tokens; now.next()) {
        copies_wait<kStagesN - 2>();
        __syncwarp();                                    // every lane's copies are there, and all are done with the unit before
        const bool known = (known_in >> stage_out) & 1u;
        fetch(position);
        position = position_ahead();
        Unit& st = queue[stage_out];
        stage_out = stage_out + 1 == kStagesN ? 0 : stage_out + 1;
        const int first = now.group * (U * kSide) + sub;
        Pair own[RUN], other[RUN];
        take_angles<RUN, INTERLEAVED, -1>(st, known, turned, l, own, other);
        T* out = dx + (now.token * heads + first) * p.dim;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool real = lane_on && first + u * kSide < heads;
            Pair g[RUN], y[RUN];
            unpack_both<T, RUN>(st.runs[4 * u][lane], st.runs[4 * u + 1][lane], real, g);
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                y[j] = mul(own[j], g[j]);
                if (turned) y[j] = fma(other[j], partner<RUN, INTERLEAVED>(g, j), y[j]);
            }
            if (weight) {
                Pair x[RUN], ss{}, dot{};
                unpack_both<T, RUN>(st.runs[4 * u + 2][lane], st.runs[4 * u + 3][lane], real, x);
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    ss = fma(x[j], x[j], ss);
                    dot = fma(mul(y[j], w[j]), x[j], dot);
                }
                const float rstd = rsqrtf(head_sum<LPH>(sum_of(ss)) * inv + p.eps);
                const float mean = head_sum<LPH>(sum_of(dot)) * rstd * inv;
                const Pair scale = pair(rstd, rstd), back = pair(-rstd * mean, -rstd * mean);
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    const Pair unit = mul(x[j], scale);
                    if (real) dw[j] = fma(y[j], unit, dw[j]);
                    y[j] = fma(unit, back, mul(mul(y[j], w[j]), scale));
                }
            }
            if (real) {
                R a, b;
                pack_both<T, RUN>(y, a, b);
                *reinterpret_cast<R*>(out + run.a) = a;
                *reinterpret_cast<R*>(out + run.b) = b;
            }
            out += kSide * p.dim;
        }
    }
    copies_wait<0>();
    if (!weight) return;
    __syncthreads();                                     // the queues are empty: their memory holds the warps' shares
    float* const share = reinterpret_cast<float*>(memory);
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
        float2 d = floats(dw[j]);
#pragma unroll
        for (int o = LPH; o < 32; o <<= 1) {
            d.x += __shfl_xor_sync(~0u, d.x, o);
            d.y += __shfl_xor_sync(~0u, d.y, o);
        }
        if (sub == 0 && lane_on)
            *reinterpret_cast<float2*>(share + warp * p.dim + (j < RUN / 2 ? run.a + 2 * j : run.b + 2 * j - RUN)) = d;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += kThreadsN) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarpsN; ++w) sum += share[w * p.dim + i];
        p.partial[int64_t(blockIdx.x) * p.dim + i] = sum;
    }
}

// The weights' gradients: sums over the blocks' shares.  blockIdx = (32 values, queries or keys); launched while the blocks still
// run.  A warp adds up every 32nd share.
template <typename T>
__global__ void __launch_bounds__(1024) weight_gradient_kernel(const __grid_constant__ NormRopeBackward p, int q_blocks, int blocks) {
    __shared__ float share[32][33];
    const bool keys = blockIdx.y != 0;
    void* const out = keys ? p.dk_weight : p.dq_weight;
    const int lo = keys ? q_blocks : 0, hi = keys ? blocks : q_blocks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = int(blockIdx.x) * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float sum = 0.f;
    if (out && i < p.dim)
#pragma unroll 8
        for (int b = lo + warp; b < hi; b += 32) sum += p.partial[int64_t(b) * p.dim + i];
    share[warp][lane] = sum;
    __syncthreads();
    sum = share[lane][warp];                              // value `warp`, share `lane`
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const int at = int(blockIdx.x) * 32 + warp;
    if (!out || lane != 0 || at >= p.dim) return;
    if (p.weights_f32) static_cast<float*>(out)[at] = sum;
    else static_cast<uint16_t*>(out)[at] = uint16_t(from_floats<T>(sum, 0.f) & 0xffffu);
}

// Blocks of an SM: what shared memory allows (228 KB, 1 KB of it per block), or registers.
template <int RUN, int LPH, int V>
constexpr int blocks_per_sm(int most) {
    const int fit = 227 * 1024 / (kWarpsN * kStagesN * int(sizeof(Stage<RUN, LPH, V>)) + 1024);
    return fit < most ? fit : most;
}
constexpr int kBackwardBlocksPerSm = blocks_per_sm<8, 16, 4 * kBackwardUnit>(kBackwardBlocks);

template <int RUN, int LPH, int V>
constexpr int queue_bytes() { return kWarpsN * kStagesN * int(sizeof(Stage<RUN, LPH, V>)); }

template <typename K>
cudaError_t with_memory(K kern, int bytes) {
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : cudaSuccess;
}

template <typename T, int RUN, int LPH>
cudaError_t forward(const NormRope& a, int num_sms, cudaStream_t stream) {
    constexpr int U = kForwardUnit, bytes = queue_bytes<RUN, LPH, 2 * U>(), per = U * (32 / LPH);
    const int q_groups = (a.q_heads + per - 1) / per, k_groups = (a.k_heads + per - 1) / per;
    const int groups = q_groups + k_groups + (a.v.data ? k_groups : 0);
    // (all that are resident, even where fewer would take as many rounds: 3 us less)
    const int64_t blocks = (a.tokens * groups + kWarpsN - 1) / kWarpsN, resident = blocks_per_sm<RUN, LPH, 2 * U>(kForwardBlocksPerSm) * num_sms;
    const unsigned grid = unsigned(blocks < resident ? blocks : resident);
    auto kern = a.interleaved ? norm_rope_kernel<T, RUN, LPH, U, true> : norm_rope_kernel<T, RUN, LPH, U, false>;
    const cudaError_t e = with_memory(kern, bytes);
    if (e != cudaSuccess) return e;
    kern<<<grid, kThreadsN, bytes, stream>>>(a, q_groups, k_groups, groups);
    return cudaGetLastError();
}

template <typename T, int RUN, int LPH>
cudaError_t backward(const NormRopeBackward& a, int num_sms, cudaStream_t stream) {
    constexpr int U = kBackwardUnit, bytes = queue_bytes<RUN, LPH, 4 * U>();
    // blocks for queries and for keys, in proportion to their units
    const int per = U * (32 / LPH), most = norm_rope_partials(num_sms);
    const int64_t q_groups = (a.q_heads + per - 1) / per, k_groups = (a.k_heads + per - 1) / per;
    auto needed = [&](int64_t groups) { const int64_t n = (a.tokens * groups + kWarpsN - 1) / kWarpsN; return n < 1 ? 1 : n; };
    int64_t q_share = most * q_groups / (q_groups + k_groups);
    q_share = q_share < 1 ? 1 : q_share > most - 1 ? most - 1 : q_share;
    const int64_t k_share = most - q_share;
    const int q_blocks = int(needed(q_groups) < q_share ? needed(q_groups) : q_share);
    const int blocks = q_blocks + int(needed(k_groups) < k_share ? needed(k_groups) : k_share);
    auto kern = a.interleaved ? norm_rope_backward_kernel<T, RUN, LPH, U, true> : norm_rope_backward_kernel<T, RUN, LPH, U, false>;
    cudaError_t e = with_memory(kern, bytes);
    if (e != cudaSuccess) return e;
    kern<<<blocks, kThreadsN, bytes, stream>>>(a, q_blocks);
    e = cudaGetLastError();
    if (e != cudaSuccess || (!a.dq_weight && !a.dk_weight)) return e;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.dim + 31) / 32, 2);
    cfg.blockDim = dim3(1024);
    cfg.stream = stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, weight_gradient_kernel<T>, a, q_blocks, blocks);
}

bool wide(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool wide(const Heads& h) { return wide(h.data) && h.token % 8 == 0 && h.head % 8 == 0; }

// Runs of eight values (16 bytes) where the layout allows, shared by as many lanes as a head needs; else runs of four and a
// warp for every head.
bool eights(int dim, int half) { return dim % 16 == 0 && half % 8 == 0; }

template <typename T>
cudaError_t forward_t(const NormRope& a, int num_sms, cudaStream_t stream) {
    const bool runs8 = eights(a.dim, a.half) && wide(a.q) && wide(a.k) && wide(a.v) && wide(a.q_out) && wide(a.k_out) && wide(a.k_cache) &&
                       wide(a.v_cache) && (a.k_page | a.k_head | a.k_slot | a.v_page | a.v_head | a.v_slot) % 8 == 0;
    if (!runs8) return forward<T, 4, 32>(a, num_sms, stream);
    return a.dim <= 64 ? forward<T, 8, 4>(a, num_sms, stream) : a.dim <= 128 ? forward<T, 8, 8>(a, num_sms, stream) : forward<T, 8, 16>(a, num_sms, stream);
}

template <typename T>
cudaError_t backward_t(const NormRopeBackward& a, int num_sms, cudaStream_t stream) {
    if (!eights(a.dim, a.half) || !wide(a.q) || !wide(a.k) || !wide(a.q_grad) || !wide(a.k_grad) || !wide(a.dq) || !wide(a.dk))
        return backward<T, 4, 32>(a, num_sms, stream);
    return a.dim <= 64 ? backward<T, 8, 4>(a, num_sms, stream) : a.dim <= 128 ? backward<T, 8, 8>(a, num_sms, stream) : backward<T, 8, 16>(a, num_sms, stream);
}

}  // namespace

int norm_rope_partials(int num_sms) { return kBackwardBlocksPerSm * num_sms; }

cudaError_t norm_rope(const NormRope& a, int num_sms, cudaStream_t stream) {
    return a.f16 ? forward_t<__half>(a, num_sms, stream) : forward_t<__nv_bfloat16>(a, num_sms, stream);
}

cudaError_t norm_rope_backward(const NormRopeBackward& a, int num_sms, cudaStream_t stream) {
    return a.f16 ? backward_t<__half>(a, num_sms, stream) : backward_t<__nv_bfloat16>(a, num_sms, stream);
}

}  // namespace dlr
