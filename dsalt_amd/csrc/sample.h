// One token a row of logits, drawn from given random numbers.
#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>

namespace dsalt {

constexpr int kSampleMaxCols = 1 << 20;

struct SampleParams {
    int rows, n_cols, dtype, u_f64;
    const void* x;
    int64_t x_st;
    const void* u;
    // a value a row, or (null) one for all
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int64_t* token;
    float* logp;
};

hipError_t sample_launch(const SampleParams& p, hipStream_t stream);

}  // namespace dsalt
