// Paged 8-bit key/value cache of a decoding step: row maps, write, read-back and the attention
// of single query tokens over it.
#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>

namespace dsalt {

constexpr int64_t kLaunchThreads = 0xffffffffll;  // a launch's threads along its first dimension

// k and v [n_blocks, n_kv, 1 << bt_log, head_dim] e4m3, scales [n_blocks, n_kv]
struct CachePages {
    int n_blocks, n_kv, bt_log, head_dim;
    uint8_t *k, *v;
    float *ks, *vs;
};

struct CacheRowsParams {
    int n_reqs, cols, bt_log, n_rows, n_pieces;
    int64_t n_free, table_st;
    const int32_t *seq_len, *new_len;
    int32_t *table, *ring;
    const int64_t* span;
    int32_t* seq_out;
    int64_t* span_out;
    int32_t *granted, *cu, *req, *pos;
    int64_t* slot;
    int32_t* pieces;
    char* ws;
};

struct CacheWriteParams {
    CachePages c;
    int n_rows, n_pieces, dtype;
    const void* k;
    int64_t k_st, k_sh;
    const void* v;
    int64_t v_st, v_sh;
    const int32_t* pieces;
};

struct CacheReadParams {
    CachePages c;
    int n_reqs, cols, n_rows, dtype;
    int64_t table_st;
    const int32_t *table, *cu, *start;
    void *k, *v;
};

struct CacheAttnParams {
    CachePages c;
    int n_rows, n_heads, n_reqs, cols, k_lmk, dtype, w_max;
    int64_t table_st;
    const void* q;
    int64_t q_st, q_sh;
    const int32_t *table, *req, *pos, *w, *lmk;
    const float* lbias;
    void* out;
    int64_t o_st, o_sh;
    float* lse;
    float scale;
    char* ws;
    size_t ws_bytes;
};

size_t cache_rows_ws_bytes(int n_reqs, int cols);
hipError_t cache_rows_launch(const CacheRowsParams& p, hipStream_t stream);
hipError_t cache_write_launch(const CacheWriteParams& p, hipStream_t stream);
hipError_t cache_read_launch(const CacheReadParams& p, hipStream_t stream);
size_t cache_attn_ws_bytes(const CacheAttnParams& p);
hipError_t cache_attn_launch(const CacheAttnParams& p, hipStream_t stream);

}  // namespace dsalt
