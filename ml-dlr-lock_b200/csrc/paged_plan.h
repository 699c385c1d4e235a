// Internal interface between the C-ABI layer and the planning kernel of the paged cache (see paged_plan.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dlr {

constexpr int kPlanMaxRequests = 8192;

struct PlanArgs {
    const int* lengths;              // (requests)
    const int* new_tokens;           // (requests)
    const unsigned char* finished;   // (requests) or null
    int* block_table;                // (requests, columns), rows table_stride apart
    int64_t table_stride;
    int columns;
    int* free_pages;                 // (pool)
    int pool;
    const int* n_free;               // (1)
    int requests, page_shift;
    int width;                       // rows of the batch per request, 0: requests lie one behind the other
    int rows;
    int* slots;                      // (rows)
    int* positions;                  // (rows)
    int* starts;                     // (requests + 1)
    int* lengths_out;                // (requests), may be lengths
    int* n_free_out;                 // (1), may be n_free
};

cudaError_t paged_plan(const PlanArgs& a, int smem_optin, cudaStream_t stream);

}  // namespace dlr
