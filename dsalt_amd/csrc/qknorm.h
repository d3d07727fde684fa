// Root-mean-square norm of each query and key head with the rotation after it, and its gradients.
#pragma once
#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

namespace dsalt {

struct QkSide {  // queries or keys: rows of `heads` heads (0: absent)
    int heads;
    const void* x;
    int64_t st, sh;
    void* y;  // forward: the output; backward: the gradient of x
    int64_t y_st, y_sh;
    const void* weight;  // [head_dim]
    const void* d;        // backward: gradient of the output
    int64_t d_st, d_sh;
    float* dw;  // backward: gradient of the weight
};

struct QkNormParams {
    int total_len, num_seqs, head_dim, dtype, w_dtype, max_pos;
    QkSide q, k;
    const int *cu, *pos;  // one of them
    const float *cos, *sin;  // [max_pos, head_dim]
    float eps;
    bool inplace;  // rows without a position keep what they hold (otherwise they become zeros)
    float* ws;
};

hipError_t qk_norm_rope_launch(const QkNormParams& p, hipStream_t stream);
size_t qk_norm_rope_bwd_ws_bytes(int total_len, int q_heads, int k_heads, int head_dim, int dtype);
hipError_t qk_norm_rope_bwd_launch(const QkNormParams& p, hipStream_t stream);

}  // namespace dsalt
