// Attention of query tokens over the paged 8-bit cache: row t is the token at position pos[t] of request
// req[t] and attends A(i) = [i - w + 1, i] U {landmarks p of its head's set : 0 <= p < i - w + 1}.
#include "cache.h"
#include "common.h"
#include "fp8.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kAttnThreads = 256;

// A block takes one row and head.  D / 16 lanes hold a key, 16 elements each; every group of lanes keeps
// its own running maximum, sum and output, joined over the block at the end.
template <typename T, int D>
__global__ __launch_bounds__(kAttnThreads) void cache_attn_kernel(CacheAttnParams p) {
    constexpr int LPK = D / 16, KPW = 64 / LPK, WAVES = kAttnThreads / 64;
    __shared__ float mls[WAVES][2];
    __shared__ float accs[WAVES][D];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int g = h / (p.n_heads / p.c.n_kv), part = lane % LPK, sub = lane / LPK;
    const int req = p.req[t], pos = p.pos[t], bt = 1 << p.c.bt_log;
    const bool live = req >= 0 && req < p.n_reqs && pos >= 0;
    const int w = max(p.w[t], 1), low = live ? max(pos - w + 1, 0) : 0;
    const int nwin = live ? pos - low + 1 : 0, nkeys = live ? nwin + p.k_lmk : 0;
    const T* qr = (const T*)p.q + (int64_t)t * p.q_st + (int64_t)h * p.q_sh + part * 16;
    float q[16], acc[16], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        q[e] = to_float(qr[e]) * p.scale;
        acc[e] = 0.f;
    }
    const int64_t set = live ? ((int64_t)h * p.n_reqs + req) * p.k_lmk : 0;
    const int32_t* table = p.table + (live ? (int64_t)req * p.table_st : 0);
    for (int i0 = wv * KPW; i0 < nkeys; i0 += WAVES * KPW) {
        const int i = i0 + sub;
        int j = -1;
        float bias = 0.f;
        if (i < nwin) {
            j = low + i;
        } else if (i < nkeys) {
            j = p.lmk[set + i - nwin];
            if (j >= low) j = -1;
            if (p.lbias) bias = p.lbias[set + i - nwin];
        }
        const int b = j >> p.c.bt_log;
        const int page = j >= 0 && b < p.cols ? table[b] : -1;
        const bool on = page >= 0 && page < p.c.n_blocks;
        u32x4 ku = {}, vu = {};
        float ks = 0.f, vs = 0.f;
        if (on) {
            const int64_t tile = (int64_t)page * p.c.n_kv + g;
            const int64_t at = ((tile << p.c.bt_log) + (j & (bt - 1))) * D + part * 16;
            ku = *(const u32x4*)(p.c.k + at);
            vu = *(const u32x4*)(p.c.v + at);
            ks = p.c.ks[tile];
            vs = p.c.vs[tile];
        }
        float f[16], s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) e4m3_x4(ku[e], f + 4 * e);
#pragma unroll
        for (int e = 0; e < 16; ++e) s += q[e] * f[e];
#pragma unroll
        for (int o = 1; o < LPK; o <<= 1) s += wave_xor(s, o);
        s = on ? s * ks + bias : -INFINITY;
        const float m1 = fmaxf(m, s), mb = m1 == -INFINITY ? 0.f : m1;
        const float a = __expf(m - mb), pr = on ? __expf(s - mb) : 0.f;
        l = l * a + pr;
#pragma unroll
        for (int e = 0; e < 4; ++e) e4m3_x4(vu[e], f + 4 * e);
        const float pv = pr * vs;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = acc[e] * a + pv * f[e];
        m = m1;
    }
    // join the wave's groups, then the waves
    float mw = m;
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1) mw = fmaxf(mw, wave_xor(mw, o));
    const float a = mw == -INFINITY ? 0.f : __expf(m - mw);
    l *= a;
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1) l += wave_xor(l, o);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        acc[e] *= a;
#pragma unroll
        for (int o = LPK; o < 64; o <<= 1) acc[e] += wave_xor(acc[e], o);
    }
    if (sub == 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) accs[wv][part * 16 + e] = acc[e];
    }
    if (lane == 0) {
        mls[wv][0] = mw;
        mls[wv][1] = l;
    }
    __syncthreads();
    if (tid < D) {
        float M = -INFINITY, L = 0.f, o = 0.f;
        for (int k = 0; k < WAVES; ++k) M = fmaxf(M, mls[k][0]);
        for (int k = 0; k < WAVES; ++k) {
            const float f = mls[k][0] == -INFINITY ? 0.f : __expf(mls[k][0] - M);
            L += mls[k][1] * f;
            o += accs[k][tid] * f;
        }
        ((T*)p.out)[(int64_t)t * p.o_st + (int64_t)h * p.o_sh + tid] = from_float<T>(L == 0.f ? 0.f : o / L);
        if (tid == 0) p.lse[(int64_t)t * p.n_heads + h] = L == 0.f ? -INFINITY : M + logf(L);
    }
}

}  // namespace

size_t cache_attn_ws_bytes(const CacheAttnParams& p) { return 0; }

hipError_t cache_attn_launch(const CacheAttnParams& p, hipStream_t stream) {
    if (p.n_rows == 0) return hipSuccess;
    const dim3 grid((unsigned)p.n_rows, (unsigned)p.n_heads);
#define RUN(T)                                                                                                        \
    if (p.c.head_dim == 128)                                                                                          \
        DSALT_LAUNCH("cache_attn", (cache_attn_kernel<T, 128>), grid, dim3(kAttnThreads), 0, stream, p);              \
    else                                                                                                              \
        DSALT_LAUNCH("cache_attn", (cache_attn_kernel<T, 64>), grid, dim3(kAttnThreads), 0, stream, p)
    switch (p.dtype) {
        case 0: RUN(float); break;
        case 1: RUN(bf16); break;
        default: RUN(f16); break;
    }
#undef RUN
    return hipGetLastError();
}

}  // namespace dsalt
