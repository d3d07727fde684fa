// Write and read-back of the paged 4-bit cache.  A token's codes and scales are its own, so that rows are written in any
// order and nothing that a page held is touched.  Both are bound by memory: 16001 rows of 8 heads of 64 in float32 (66 MB, 9 MB
// of them as held) are written in 13 us and read back in 18 us, 256 rows of 2 heads of 128 in bfloat16 in 3 and 4 us.
#include <algorithm>

#include "cache4.h"
#include "common.h"
#include "fp4.h"
#include "timing.h"

namespace dsalt {

namespace {

template <typename T>
__device__ __forceinline__ void load8(const T* x, float* f) {
    typedef T vec __attribute__((ext_vector_type(8), aligned(16)));
    const vec v = *(const vec*)x;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_float(v[e]);
}

// maximum over the four lanes that share lane / 4
__device__ __forceinline__ uint32_t max_of4(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));  // lanes 1, 0, 3, 2
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));  // 2, 3, 0, 1
}

// ---------------------------------------------------------------------- write
// gridDim.y blocks take a piece (rows of one request within one page); a thread eight elements of a row and head, four threads the
// 32 of a scale.  Magnitudes are compared as the integers of their bits, in
// which everything not finite lies at the infinity or above.
template <typename T>
__global__ __launch_bounds__(256) void cache4_write_kernel(Cache4WriteParams p) {
    const int4 piece = ((const int4*)p.pieces)[blockIdx.x];
    const int row0 = piece.x, rows = piece.y, page = piece.z, off = piece.w;
    const int bt = 1 << p.c.bt_log, D = p.c.head_dim, per_log = __builtin_ctz(D / 8), G = p.c.n_kv;
    // pieces past the last (no rows), and any that does not lie within the rows and one page
    if (rows <= 0 || row0 < 0 || rows > p.n_rows - row0 || page < 0 || page >= p.c.n_blocks || off < 0 || rows > bt - off) return;
    const int heads = 2 * G;  // keys, then values
    const int n = (rows * heads) << per_log;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < n; i += gridDim.y * 256) {
        const int c = i & ((1 << per_log) - 1), rh = i >> per_log, r = rh / heads, h = rh - r * heads;
        const int val = h >= G, g = h - val * G;
        const T* x = val ? (const T*)p.v + (int64_t)(row0 + r) * p.v_st + (int64_t)g * p.v_sh
                         : (const T*)p.k + (int64_t)(row0 + r) * p.k_st + (int64_t)g * p.k_sh;
        float f[8];
        load8(x + c * 8, f);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
        top = max_of4(top);
        const bool held = top < 0x7f800000u;  // all finite
        const uint32_t exponent = held ? e8m0_of(__uint_as_float(top)) : 255u;
        const int64_t token = ((((int64_t)page * G + g) << p.c.bt_log) + off + r) * 2 + val;
        *(uint32_t*)(p.c.kv + token * (D / 2) + c * 4) = held ? to_e2m1_x8(f, e8m0(exponent)) : 0u;
        if ((c & 3) == 0) p.c.scale[token * (D / 32) + (c >> 2)] = (uint8_t)exponent;
    }
}

// ----------------------------------------------------------------------- read
// Row t of a packed batch is token start[r] + t - cu[r] of its request r.  A thread takes eight elements of one head,
// keys and values.
template <typename T>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache4ReadParams p) {
    typedef T vec __attribute__((ext_vector_type(8), aligned(16)));
    const int D = p.c.head_dim, per = p.c.n_kv * (D / 8);
    const int64_t n = (int64_t)p.n_rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int t = (int)(i / per), x = (int)(i - (int64_t)t * per), g = x / (D / 8), c = x - g * (D / 8);
        int lo = 0, hi = p.n_reqs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid + 1] > t) hi = mid;
            else lo = mid + 1;
        }
        vec k = {}, v = {};
        if (lo < p.n_reqs && t >= p.cu[lo]) {
            const int64_t pos = (int64_t)(p.start ? p.start[lo] : 0) + t - p.cu[lo];
            const int64_t b = pos >> p.c.bt_log;
            const int page = pos >= 0 && b < p.cols ? p.table[lo * p.table_st + b] : -1;
            if (page >= 0 && page < p.c.n_blocks) {
                const int64_t token = (((int64_t)page * p.c.n_kv + g) << p.c.bt_log) + (pos & ((1 << p.c.bt_log) - 1));
                const uint8_t* codes = p.c.kv + token * D + c * 4;
                const uint8_t* exps = p.c.scale + token * (D / 16) + (c >> 2);
                const uint32_t ku = *(const uint32_t*)codes, vu = *(const uint32_t*)(codes + D / 2);
                const float ks = e8m0(exps[0]), vs = e8m0(exps[D / 32]);
                float f[8];
                e2m1_x8(ku, ks, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = from_float<T>(f[e]);
                e2m1_x8(vu, vs, f);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = from_float<T>(f[e]);
            }
        }
        *(vec*)((T*)p.k + ((int64_t)t * p.c.n_kv + g) * D + c * 8) = k;
        *(vec*)((T*)p.v + ((int64_t)t * p.c.n_kv + g) * D + c * 8) = v;
    }
}

// As many blocks to a piece as give each thread eight elements of an average piece, up to sixteen.  (Write and read of the 16001
// rows with one block to a piece 37.9 us, four 34.9, sixteen 33.7; pieces of single rows, which have work for one, take 6.1 with
// any number.)
template <typename T>
void write_pieces(const Cache4WriteParams& p, hipStream_t stream) {
    const int64_t threads = (int64_t)p.n_rows * 2 * p.c.n_kv * (p.c.head_dim / 8) / p.n_pieces;
    const unsigned parts = (unsigned)std::max(std::min((threads + 255) / 256, (int64_t)16), (int64_t)1);
    Cache4WriteParams s = p;
    for (int64_t k = 0; k < p.n_pieces; k += s.n_pieces) {
        s.n_pieces = (int)std::min(p.n_pieces - k, kLaunchThreads / 256);
        s.pieces = p.pieces + 4 * k;
        DSALT_LAUNCH("cache4_write", cache4_write_kernel<T>, dim3((unsigned)s.n_pieces, parts), dim3(256), 0, stream, s);
    }
}

}  // namespace

hipError_t cache4_write_launch(const Cache4WriteParams& p, hipStream_t stream) {
    if (p.n_pieces == 0 || p.n_rows == 0) return hipSuccess;
    switch (p.dtype) {
        case 0: write_pieces<float>(p, stream); break;
        case 1: write_pieces<bf16>(p, stream); break;
        default: write_pieces<f16>(p, stream); break;
    }
    return hipGetLastError();
}

hipError_t cache4_read_launch(const Cache4ReadParams& p, hipStream_t stream) {
    if (p.n_rows == 0) return hipSuccess;
    const int64_t n = (int64_t)p.n_rows * p.c.n_kv * (p.c.head_dim / 8);
    const dim3 grid((unsigned)std::min((n + 255) / 256, (int64_t)1 << 20));
    switch (p.dtype) {
        case 0: DSALT_LAUNCH("cache4_read", cache4_read_kernel<float>, grid, dim3(256), 0, stream, p); break;
        case 1: DSALT_LAUNCH("cache4_read", cache4_read_kernel<bf16>, grid, dim3(256), 0, stream, p); break;
        default: DSALT_LAUNCH("cache4_read", cache4_read_kernel<f16>, grid, dim3(256), 0, stream, p); break;
    }
    return hipGetLastError();
}

}  // namespace dsalt
