// Drafted tokens taken or refused against the target's probabilities.
#pragma once
#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

namespace dsalt {

struct VerifyParams {
    int n_reqs, n_rows, n_cols, dtype, u_f64;
    const void* x;  // target logits
    int64_t x_st;
    const void* y;  // draft logits, or null: drafts certain of themselves
    int64_t y_st;
    const int64_t* tokens;
    const int32_t* cu;
    const void *u, *v;
    // a value a request, or (null) one for all
    const float *temperature, *draft_temperature;
    float temperature_all, draft_temperature_all;
    int32_t* accepted;
    int64_t* out;
    char* ws;
};

size_t verify_ws_bytes(const VerifyParams& p);
hipError_t verify_launch(const VerifyParams& p, hipStream_t stream);

}  // namespace dsalt
