// Drawing the next token of each row.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sg {

struct SampleTokens {
    const void* logits;          // [B, V], rows row_stride elements apart
    int64_t row_stride;
    int type;                    // 0 bf16, 1 fp16, 3 fp32
    int B, V;
    const float* u;              // [B] in [0, 1)
    // one value a row, or null: the value for all rows
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int* token;                  // [B]
    float* logprob;              // [B]
};
const char* sample_tokens(const SampleTokens& p, int num_sms, cudaStream_t s);

}  // namespace sg
