// RMS norm of every query and key head with the rotation by position in the same pass, its gradient, and the form that puts
// keys and values straight into a paged cache.
//
//   n = x * rsqrt(mean(x^2) + eps) * w             (left out where there is no weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)       over the pairs of the first 2 * half values; the rest passes through
//
// Pairs are (i, i + half), or (2i, 2i + 1) where the layout is interleaved.  Backward, with g the incoming gradient turned
// back by the same angle, u = x * rstd:   dx = rstd * (g w - u * mean(g w u)),   dw = sum of g u over tokens and heads.
//
// Bound by memory: every value is read once and written once.  dim / 8 lanes share a head and each holds two runs of four
// values that are each other's partners (runs l and l + half / 4, or neighbouring ones), so that the rotation needs no
// exchange between lanes, and a lane needs 4 cosines and 4 sines instead of 8 of each.  A warp takes several heads of one
// token, which share those.  Everything between the load and the store is fp32, rounded once.
#include "norm_rope.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace dlr {

namespace {

constexpr int kThreadsN = 256;
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

template <typename T>
__device__ __forceinline__ void unpack(uint2 v, float (&f)[4]) {
    const float2 lo = to_float2<T>(v.x), hi = to_float2<T>(v.y);
    f[0] = lo.x, f[1] = lo.y, f[2] = hi.x, f[3] = hi.y;
}
template <typename T>
__device__ __forceinline__ uint2 pack(const float (&f)[4]) {
    return make_uint2(from_floats<T>(f[0], f[1]), from_floats<T>(f[2], f[3]));
}

// the two runs of four values that lane l of a head holds, as indexes of values
struct Runs {
    int a, b;
    bool turned;
};

template <bool INTERLEAVED>
__device__ __forceinline__ Runs runs_of(int l, int half) {
    Runs r;
    r.turned = l < half / 4;
    if (INTERLEAVED || !r.turned) {
        r.a = 8 * l;
        r.b = 8 * l + 4;
    } else {
        r.a = 4 * l;
        r.b = 4 * l + half;
    }
    return r;
}

// sign = 1: by the angle; -1: back
template <bool INTERLEAVED>
__device__ __forceinline__ void turn(float (&a)[4], float (&b)[4], const float (&c)[4], const float (&s)[4]) {
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
            a[2 * i] = x * c[i] - y * s[i];
            a[2 * i + 1] = y * c[i] + x * s[i];
            b[2 * i] = z * c[2 + i] - w * s[2 + i];
            b[2 * i + 1] = w * c[2 + i] + z * s[2 + i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * c[i] - y * s[i];
            b[i] = y * c[i] + x * s[i];
        }
    }
}

__device__ __forceinline__ void load4(const float* p, float (&f)[4]) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}

template <typename T>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int at, float (&f)[4]) {
    if (f32) load4(static_cast<const float*>(w) + at, f);
    else unpack<T>(__ldg(reinterpret_cast<const uint2*>(static_cast<const T*>(w) + at)), f);
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

// cosines and sines of this lane's pairs; a position outside the tables gives NaN
template <int SIGN>
__device__ __forceinline__ bool angles(const float* cos, const float* sin, int half, int rows, int64_t position, bool turned, int l,
                                       float (&c)[4], float (&s)[4]) {
    const bool known = position >= 0 && position < rows;
    if (turned && known) {
        load4(cos + position * half + 4 * l, c);
        load4(sin + position * half + 4 * l, s);
        if (SIGN < 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = -s[i];
    }
    return known;
}

// A warp: one token, up to U * 32 / LPH heads of its queries, keys or values.
template <typename T, int LPH, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreadsN) norm_rope_kernel(const __grid_constant__ NormRope p, int q_groups, int k_groups, int groups) {
    constexpr int kSide = 32 / LPH;                      // heads side by side in a warp
    const int lane = threadIdx.x & 31, l = lane % LPH, sub = lane / LPH;
    const int64_t unit = int64_t(blockIdx.x) * kWarpsN + (threadIdx.x >> 5);
    const int64_t token = unit / groups;
    if (token >= p.tokens) return;
    int group = int(unit - token * groups);
    int kind = 0;
    if (group >= q_groups) {
        group -= q_groups;
        kind = 1;
        if (group >= k_groups) {
            group -= k_groups;
            kind = 2;
        }
    }
    const Heads& in = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const int heads = kind == 0 ? p.q_heads : p.k_heads;
    const int first = group * (U * kSide) + sub;

    // rows of heads that this warp writes: q_out or k_out, and the token's slot of the cache
    T* const out = kind == 0 ? static_cast<T*>(p.q_out) + token * p.q_heads * p.dim
                   : kind == 1 && p.k_out ? static_cast<T*>(p.k_out) + token * p.k_heads * p.dim : nullptr;
    T* cached = nullptr;
    int64_t cached_head = 0;
    if (kind != 0 && p.slots) {
        const int64_t slot = p.slots[token];
        if (slot >= 0 && slot < p.n_slots) {             // (a row without a place in the cache otherwise)
            const int64_t page = slot >> p.page_shift, at = slot & ((1 << p.page_shift) - 1);
            cached = kind == 1 ? static_cast<T*>(p.k_cache) + page * p.k_page + at * p.k_slot
                               : static_cast<T*>(p.v_cache) + page * p.v_page + at * p.v_slot;
            cached_head = kind == 1 ? p.k_head : p.v_head;
        }
    }
    if (!out && !cached) return;
    auto store = [&](int h, const Runs& run, uint2 a, uint2 b) {
        if (out) {
            *reinterpret_cast<uint2*>(out + h * p.dim + run.a) = a;
            *reinterpret_cast<uint2*>(out + h * p.dim + run.b) = b;
        }
        if (cached) {
            *reinterpret_cast<uint2*>(cached + h * cached_head + run.a) = a;
            *reinterpret_cast<uint2*>(cached + h * cached_head + run.b) = b;
        }
    };

    const Runs run = runs_of<INTERLEAVED>(l, p.half);
    const bool lane_on = 8 * l < p.dim;
    const T* x = static_cast<const T*>(in.data) + token * in.token;
    uint2 va[U], vb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = first + u * kSide;
        va[u] = vb[u] = make_uint2(0, 0);
        if (lane_on && h < heads) {
            va[u] = *reinterpret_cast<const uint2*>(x + h * in.head + run.a);
            vb[u] = *reinterpret_cast<const uint2*>(x + h * in.head + run.b);
        }
    }
    if (kind == 2) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = first + u * kSide;
            if (lane_on && h < heads) store(h, run, va[u], vb[u]);
        }
        return;
    }
    float c[4], s[4], wa[4], wb[4];
    const void* weight = kind == 0 ? p.q_weight : p.k_weight;
    const bool known = angles<1>(p.cos, p.sin, p.half, p.table_rows, position_of(p.positions, p.positions_64, token), run.turned && lane_on, l, c, s);
    if (weight && lane_on) {
        load_weight<T>(weight, p.weights_f32, run.a, wa);
        load_weight<T>(weight, p.weights_f32, run.b, wb);
    }
    const float inv = 1.0f / float(p.dim);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float a[4], b[4];
        unpack<T>(va[u], a);
        unpack<T>(vb[u], b);
        if (weight) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
            const float rstd = rsqrtf(head_sum<LPH>(ss) * inv + p.eps);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] *= rstd * wa[i];
                b[i] *= rstd * wb[i];
            }
        }
        if (run.turned) turn<INTERLEAVED>(a, b, c, s);
        if (!known)
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = b[i] = __int_as_float(0x7fffffff);
        const int h = first + u * kSide;
        if (lane_on && h < heads) store(h, run, pack<T>(a), pack<T>(b));
    }
}

// Blocks of the first q_blocks take query heads, the others key heads; a warp walks over (token, group of heads) and keeps
// its share of the weight's gradient in registers.  Shares are added up in a fixed order: shuffles, the block's warps, and
// (weight_gradient_kernel) the blocks, so that results repeat bit for bit.
template <typename T, int LPH, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreadsN) norm_rope_backward_kernel(const __grid_constant__ NormRopeBackward p, int q_blocks) {
    constexpr int kSide = 32 / LPH;
    __shared__ float share[kWarpsN][LPH * 8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPH, sub = lane / LPH;
    const bool keys = int(blockIdx.x) >= q_blocks;
    const int block = keys ? int(blockIdx.x) - q_blocks : int(blockIdx.x), blocks = keys ? int(gridDim.x) - q_blocks : q_blocks;
    const Heads& in = keys ? p.k : p.q;
    const Heads& grad = keys ? p.k_grad : p.q_grad;
    const void* weight = keys ? p.k_weight : p.q_weight;
    T* const dx = static_cast<T*>(keys ? p.dk : p.dq);
    const int heads = keys ? p.k_heads : p.q_heads, groups = (heads + U * kSide - 1) / (U * kSide);
    const Runs run = runs_of<INTERLEAVED>(l, p.half);
    const bool lane_on = 8 * l < p.dim;
    float wa[4] = {}, wb[4] = {}, da[4] = {}, db[4] = {};
    if (weight && lane_on) {
        load_weight<T>(weight, p.weights_f32, run.a, wa);
        load_weight<T>(weight, p.weights_f32, run.b, wb);
    }
    const float inv = 1.0f / float(p.dim);
    const int64_t units = p.tokens * groups;
    for (int64_t unit = int64_t(block) * kWarpsN + warp; unit < units; unit += int64_t(blocks) * kWarpsN) {
        const int64_t token = unit / groups;
        const int first = int(unit - token * groups) * (U * kSide) + sub;
        const T* x = static_cast<const T*>(in.data) + token * in.token;
        const T* g = static_cast<const T*>(grad.data) + token * grad.token;
        uint2 xa[U], xb[U], ga[U], gb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = first + u * kSide;
            xa[u] = xb[u] = ga[u] = gb[u] = make_uint2(0, 0);
            if (lane_on && h < heads) {
                ga[u] = *reinterpret_cast<const uint2*>(g + h * grad.head + run.a);
                gb[u] = *reinterpret_cast<const uint2*>(g + h * grad.head + run.b);
                if (weight) {
                    xa[u] = *reinterpret_cast<const uint2*>(x + h * in.head + run.a);
                    xb[u] = *reinterpret_cast<const uint2*>(x + h * in.head + run.b);
                }
            }
        }
        float c[4], s[4];
        const bool known = angles<-1>(p.cos, p.sin, p.half, p.table_rows, position_of(p.positions, p.positions_64, token), run.turned && lane_on, l, c, s);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float a[4], b[4];
            unpack<T>(ga[u], a);
            unpack<T>(gb[u], b);
            if (run.turned) turn<INTERLEAVED>(a, b, c, s);
            if (!known)
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = b[i] = __int_as_float(0x7fffffff);
            if (weight) {
                float ua[4], ub[4], ss = 0.f, dot = 0.f;
                unpack<T>(xa[u], ua);
                unpack<T>(xb[u], ub);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ss += ua[i] * ua[i] + ub[i] * ub[i];
                    dot += a[i] * wa[i] * ua[i] + b[i] * wb[i] * ub[i];
                }
                const float rstd = rsqrtf(head_sum<LPH>(ss) * inv + p.eps);
                const float mean = head_sum<LPH>(dot) * rstd * inv;
                const bool real = first + u * kSide < heads;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ua[i] *= rstd;
                    ub[i] *= rstd;
                    if (real) {
                        da[i] += a[i] * ua[i];
                        db[i] += b[i] * ub[i];
                    }
                    a[i] = rstd * (a[i] * wa[i] - ua[i] * mean);
                    b[i] = rstd * (b[i] * wb[i] - ub[i] * mean);
                }
            }
            const int h = first + u * kSide;
            if (lane_on && h < heads) {
                T* out = dx + (token * heads + h) * p.dim;
                *reinterpret_cast<uint2*>(out + run.a) = pack<T>(a);
                *reinterpret_cast<uint2*>(out + run.b) = pack<T>(b);
            }
        }
    }
    if (!weight) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = LPH; o < 32; o <<= 1) {
            da[i] += __shfl_xor_sync(~0u, da[i], o);
            db[i] += __shfl_xor_sync(~0u, db[i], o);
        }
        if (sub == 0 && lane_on) {
            share[warp][run.a + i] = da[i];
            share[warp][run.b + i] = db[i];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += kThreadsN) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarpsN; ++w) sum += share[w][i];
        p.partial[int64_t(blockIdx.x) * p.dim + i] = sum;
    }
}

// block 0: queries, 1: keys
template <typename T>
__global__ void __launch_bounds__(1024) weight_gradient_kernel(const __grid_constant__ NormRopeBackward p, int q_blocks, int blocks) {
    __shared__ float share[1024];
    const bool keys = blockIdx.x != 0;
    void* const out = keys ? p.dk_weight : p.dq_weight;
    if (!out) return;
    const int lo = keys ? q_blocks : 0, hi = keys ? blocks : q_blocks;
    const int parts = 1024 / p.dim, part = int(threadIdx.x) / p.dim, i = int(threadIdx.x) % p.dim;
    float sum = 0.f;
    if (part < parts)
        for (int b = lo + part; b < hi; b += parts) sum += p.partial[int64_t(b) * p.dim + i];
    share[threadIdx.x] = sum;
    __syncthreads();
    if (part != 0) return;
    for (int k = 1; k < parts; ++k) sum += share[k * p.dim + i];
    if (p.weights_f32) static_cast<float*>(out)[i] = sum;
    else static_cast<uint16_t*>(out)[i] = uint16_t(from_floats<T>(sum, 0.f) & 0xffffu);
}

constexpr int kBlocksPerSm = 4;

template <typename T, int LPH, int U>
cudaError_t forward_u(const NormRope& a, cudaStream_t stream) {
    const int per = U * (32 / LPH);
    const int q_groups = (a.q_heads + per - 1) / per, k_groups = (a.k_heads + per - 1) / per;
    const int groups = q_groups + k_groups + (a.v.data ? k_groups : 0);
    const int64_t grid = (a.tokens * groups + kWarpsN - 1) / kWarpsN;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    if (a.interleaved) norm_rope_kernel<T, LPH, U, true><<<unsigned(grid), kThreadsN, 0, stream>>>(a, q_groups, k_groups, groups);
    else norm_rope_kernel<T, LPH, U, false><<<unsigned(grid), kThreadsN, 0, stream>>>(a, q_groups, k_groups, groups);
    return cudaGetLastError();
}

template <typename T, int LPH>
cudaError_t forward(const NormRope& a, cudaStream_t stream) {
    return forward_u<T, LPH, 4>(a, stream);
}

template <typename T, int LPH>
cudaError_t backward(const NormRopeBackward& a, int num_sms, cudaStream_t stream) {
    constexpr int U = 2;
    const int blocks = norm_rope_partials(num_sms);
    int q_blocks = int(int64_t(blocks) * a.q_heads / (a.q_heads + a.k_heads));
    if (q_blocks < 1) q_blocks = 1;
    if (q_blocks > blocks - 1) q_blocks = blocks - 1;
    if (a.interleaved) norm_rope_backward_kernel<T, LPH, U, true><<<blocks, kThreadsN, 0, stream>>>(a, q_blocks);
    else norm_rope_backward_kernel<T, LPH, U, false><<<blocks, kThreadsN, 0, stream>>>(a, q_blocks);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || (!a.dq_weight && !a.dk_weight)) return e;
    weight_gradient_kernel<T><<<2, 1024, 0, stream>>>(a, q_blocks, blocks);
    return cudaGetLastError();
}

}  // namespace

int norm_rope_partials(int num_sms) { return kBlocksPerSm * num_sms; }

cudaError_t norm_rope(const NormRope& a, cudaStream_t stream) {
    if (a.dim <= 64) return a.f16 ? forward<__half, 8>(a, stream) : forward<__nv_bfloat16, 8>(a, stream);
    if (a.dim <= 128) return a.f16 ? forward<__half, 16>(a, stream) : forward<__nv_bfloat16, 16>(a, stream);
    return a.f16 ? forward<__half, 32>(a, stream) : forward<__nv_bfloat16, 32>(a, stream);
}

cudaError_t norm_rope_backward(const NormRopeBackward& a, int num_sms, cudaStream_t stream) {
    if (a.dim <= 64) return a.f16 ? backward<__half, 8>(a, num_sms, stream) : backward<__nv_bfloat16, 8>(a, num_sms, stream);
    if (a.dim <= 128) return a.f16 ? backward<__half, 16>(a, num_sms, stream) : backward<__nv_bfloat16, 16>(a, num_sms, stream);
    return a.f16 ? backward<__half, 32>(a, num_sms, stream) : backward<__nv_bfloat16, 32>(a, num_sms, stream);
}

}  // namespace dlr
