// Internal interface between the C-ABI layer and the norm-and-rotation kernels (see norm_rope.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dlr {

// a (tokens, heads, dim) tensor of 16-bit values, strides in elements, dim contiguous
struct Heads {
    const void* data;
    int64_t token, head;
};

struct NormRope {
    Heads q, k, v;                       // v: for the append only (null data otherwise)
    const void* q_weight;                // (dim) or null: no norm
    const void* k_weight;
    const float* cos;                    // (table_rows, half)
    const float* sin;
    const void* positions;               // (tokens)
    void* q_out;                         // (tokens, q_heads, dim) contiguous
    void* k_out;                         // the same, or null
    const int* slots;                    // (tokens): k and v go to the cache (k to k_out too, if there is one); or null
    void* k_cache;                       // (pages, k_heads, page tokens, dim), strides in elements
    void* v_cache;
    int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
    int64_t n_slots;
    int page_shift;
    int64_t tokens;
    int q_heads, k_heads, dim, half, table_rows;
    bool f16, weights_f32, positions_64, interleaved;
    float eps;
};

struct NormRopeBackward {
    Heads q, k;                          // the inputs of the forward (unused without a norm)
    Heads q_grad, k_grad;                // gradients of its outputs
    const void* q_weight;
    const void* k_weight;
    const float* cos;
    const float* sin;
    const void* positions;
    void* dq;                            // contiguous
    void* dk;
    void* dq_weight;                     // (dim), in the type of the weights, or null
    void* dk_weight;
    float* partial;                      // norm_rope_partials() x dim, with a norm
    int64_t tokens;
    int q_heads, k_heads, dim, half, table_rows;
    bool f16, weights_f32, positions_64, interleaved;
    float eps;
};

int norm_rope_partials(int num_sms);
cudaError_t norm_rope(const NormRope& a, int num_sms, cudaStream_t stream);
cudaError_t norm_rope_backward(const NormRopeBackward& a, int num_sms, cudaStream_t stream);

}  // namespace dlr
