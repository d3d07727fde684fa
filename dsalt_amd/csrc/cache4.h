// Paged 4-bit key/value cache: write, read-back and the attention of query tokens over it.
#pragma once
#include "cache.h"

namespace dsalt {

// A token of a head: `kv` [n_blocks, n_kv, 1 << bt_log, 2, head_dim / 2] e2m1 codes, two a byte, the key's before the
// value's, and `scale` [n_blocks, n_kv, 1 << bt_log, 2, head_dim / 32], the exponent (above -127) of a power of two for
// each 32 elements.
struct Cache4Pages {
    int n_blocks, n_kv, bt_log, head_dim;
    uint8_t *kv, *scale;
};

struct Cache4WriteParams {
    Cache4Pages c;
    int n_rows, n_pieces, dtype;
    const void* k;
    int64_t k_st, k_sh;
    const void* v;
    int64_t v_st, v_sh;
    const int32_t* pieces;
};

struct Cache4ReadParams {
    Cache4Pages c;
    int n_reqs, cols, n_rows, dtype;
    int64_t table_st;
    const int32_t *table, *cu, *start;
    void *k, *v;
};

struct Cache4AttnParams {
    Cache4Pages c;
    int n_rows, n_heads, n_reqs, cols, k_lmk, dtype, w_max, per;  // per: rows of a request that lie side by side
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
};

hipError_t cache4_write_launch(const Cache4WriteParams& p, hipStream_t stream);
hipError_t cache4_read_launch(const Cache4ReadParams& p, hipStream_t stream);
size_t cache4_attn_ws_bytes(const Cache4AttnParams& p);
hipError_t cache4_attn_launch(const Cache4AttnParams& p, hipStream_t stream);

}  // namespace dsalt
