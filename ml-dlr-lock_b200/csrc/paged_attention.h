// Internal interface between the C-ABI layer and the paged attention kernels (see paged_attention.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace dlr {

struct PagedAttention {
    const void* q;                       // (requests, heads, dim), strides in elements, dim contiguous
    int64_t q_request, q_head;
    const void* k_cache;                 // (pages, kv_heads, page tokens, dim), strides in elements, dim contiguous
    const void* v_cache;
    int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
    const int* block_table;              // (requests, columns), rows table_stride apart
    int64_t table_stride;
    const int* lengths;                  // (requests)
    void* out;                           // (requests, heads, dim) contiguous
    void* workspace;
    int requests, heads, kv_heads, dim, columns, page_shift, pages;
    bool f16;
    float scale;
};

bool paged_attention_supported(int heads, int kv_heads, int dim);
size_t paged_attention_workspace_bytes(int heads, int kv_heads, int dim, int num_sms);
cudaError_t paged_attention(const PagedAttention& a, int num_sms, cudaStream_t stream);

}  // namespace dlr
