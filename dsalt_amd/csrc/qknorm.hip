// A root-mean-square norm of every query and key head and the half-split rotation after it, in one pass, and the
// gradients of both.  For a head x of D elements at position p, halves indexed by j < D/2:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w
//   y1[j] = n1[j] cos[p][j] - n2[j] sin[p][j],  y2[j] = n2[j] cos[p][D/2 + j] + n1[j] sin[p][D/2 + j]
// and with d the gradient of y:
//   dn1 = d1 cos1 + d2 sin2,  dn2 = d2 cos2 - d1 sin1,  dw = sum over rows and heads of dn x r,
//   dx = r (w dn) - x r^3 mean(w dn x)
// All in float32, rounded once when stored.  Bound by memory: the forward reads and writes every element once, the
// backward reads two and writes one.
//
// D/16 lanes take a head (rounded up to a power of two), each eight elements of either half, so that both partners of
// the rotation lie in one lane and the norm's sum crosses a few lanes only.  A wave takes 64 / lanes tokens at a time and some
// of their heads, one after the other, always of the same side: weights are read once, cosines and sines once a token, and the
// first head's elements are asked for before its position is looked up.  The weights' gradients stay in registers over all that
// a wave takes, are joined over the block and then, in the order of the blocks, by a second kernel: no atomics, the same bits
// in every run.  At 32768 tokens of 16 and 2 heads of 128 in bfloat16 the forward moves its 302 MB (and 34 MB of cosines and
// sines) in 70 us, the backward its 453 MB in 100 us.  At 16001 tokens of 16 and 16 heads of 64 the backward takes 50 us: 38 in its
// kernel, 4 in the second and the rest between the two.
#include <algorithm>

#include "common.h"
#include "qknorm.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

template <typename T> struct Eight { typedef T type __attribute__((ext_vector_type(8), aligned(16))); };
typedef float f32x8 __attribute__((ext_vector_type(8), aligned(16)));

// sum over the LP lanes that share lane / LP
template <int LP>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
    for (int o = 1; o < LP; o <<= 1) v += wave_xor(v, o);
    return v;
}

// eight elements of a weight from j
__device__ __forceinline__ f32x8 weight8(const QkNormParams& p, const void* w, int j) {
    f32x8 o;
    if (p.w_dtype == 0) return *(const f32x8*)((const float*)w + j);
    if (p.w_dtype == 1) {
        const typename Eight<bf16>::type v = *(const typename Eight<bf16>::type*)((const bf16*)w + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = to_float(v[e]);
    } else {
        const typename Eight<f16>::type v = *(const typename Eight<f16>::type*)((const f16*)w + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = to_float(v[e]);
    }
    return o;
}

// position of row t: given, or its place in the sequence that holds it; -1 outside the sequences and the tables
__device__ __forceinline__ int position(const QkNormParams& p, int t) {
    int at = -1;
    if (p.pos) {
        at = p.pos[t];
    } else if (t >= p.cu[0] && t < p.cu[p.num_seqs]) {
        int lo = 0, hi = p.num_seqs - 1;  // the last sequence that begins at t or before
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (p.cu[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        at = t - p.cu[lo];
    }
    return at >= 0 && at < p.max_pos ? at : -1;
}

// how the work is cut: a wave takes up to q_heads heads of the queries or k_heads of the keys, of every `lines`-th group of
// 64 / LP tokens
struct QkPlan {
    int q_heads, k_heads, q_chunks, chunks, lines, blocks;
};

// the heads that a wave takes (side 1: keys); false for a wave left over
struct QkWave {
    int side, first, last, line;
};

__device__ __forceinline__ bool wave_part(const QkNormParams& p, const QkPlan& a, QkWave& w) {
    const int at = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + (int)(threadIdx.x >> 6)), chunk = at % a.chunks;
    w.line = at / a.chunks;
    w.side = chunk >= a.q_chunks;
    w.first = w.side ? (chunk - a.q_chunks) * a.k_heads : chunk * a.q_heads;
    w.last = w.side ? min(w.first + a.k_heads, p.k.heads) : min(w.first + a.q_heads, p.q.heads);
    return w.line < a.lines;
}

template <typename T, int LP>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(QkNormParams p, QkPlan a) {
    typedef typename Eight<T>::type vec8;
    constexpr int TOK = 64 / LP;
    const int lane = threadIdx.x & 63, part = lane % LP, sub = lane / LP, half = p.head_dim >> 1, j0 = part * 8;
    const float inv_d = 1.f / (float)p.head_dim;
    QkWave w;
    if (!wave_part(p, a, w)) return;
    const QkSide x = w.side ? p.k : p.q;
    f32x8 w1 = {}, w2 = {};
    if (j0 < half) {
        w1 = weight8(p, x.weight, j0);
        w2 = weight8(p, x.weight, half + j0);
    }
    for (int64_t t0 = (int64_t)w.line * TOK; t0 < p.total_len; t0 += (int64_t)a.lines * TOK) {
        const bool row = t0 + sub < p.total_len, on = row && j0 < half;
        const int t = row ? (int)t0 + sub : 0;
        const T* in = (const T*)x.x + (int64_t)t * x.st + j0;
        T* out = (T*)x.y + (int64_t)t * x.y_st + j0;
        vec8 a1 = {}, a2 = {};
        auto load = [&](int h, vec8& v1, vec8& v2) {
            if (on) {
                v1 = *(const vec8*)(in + (int64_t)h * x.sh);
                v2 = *(const vec8*)(in + (int64_t)h * x.sh + half);
            }
        };
        load(w.first, a1, a2);
        const int pos = row ? position(p, t) : -1;
        // n cos and n sin with the weight taken into them
        f32x8 w1c = {}, w2s = {}, w2c = {}, w1s = {};
        if (on && pos >= 0) {
            const int64_t at = (int64_t)pos * p.head_dim + j0;
            w1c = w1 * *(const f32x8*)(p.cos + at);
            w2c = w2 * *(const f32x8*)(p.cos + at + half);
            w2s = w2 * *(const f32x8*)(p.sin + at);
            w1s = w1 * *(const f32x8*)(p.sin + at + half);
        }
        for (int h = w.first; h < w.last; ++h) {
            vec8 n1 = {}, n2 = {};
            if (h + 1 < w.last) load(h + 1, n1, n2);
            float f1[8], f2[8], ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f1[e] = to_float(a1[e]);
                f2[e] = to_float(a2[e]);
                ss += f1[e] * f1[e] + f2[e] * f2[e];
            }
            const float r = 1.f / sqrtf(sum_lanes<LP>(ss) * inv_d + p.eps);
            vec8 o1, o2;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                o1[e] = from_float<T>(pos < 0 ? 0.f : r * (f1[e] * w1c[e] - f2[e] * w2s[e]));
                o2[e] = from_float<T>(pos < 0 ? 0.f : r * (f2[e] * w2c[e] + f1[e] * w1s[e]));
            }
            if (on && (pos >= 0 || !p.inplace)) {
                *(vec8*)(out + (int64_t)h * x.y_sh) = o1;
                *(vec8*)(out + (int64_t)h * x.y_sh + half) = o2;
            }
            a1 = n1;
            a2 = n2;
        }
    }
}

template <typename T, int LP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2) void qk_norm_rope_bwd_kernel(QkNormParams p, QkPlan a) {
    typedef typename Eight<T>::type vec8;
    constexpr int TOK = 64 / LP;
    __shared__ float sums[kWaves][LP * 16];
    __shared__ int side_of[kWaves];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, part = lane % LP, sub = lane / LP, half = p.head_dim >> 1, j0 = part * 8;
    const float inv_d = 1.f / (float)p.head_dim;
    QkWave w;
    const bool mine = wave_part(p, a, w);
    const QkSide x = w.side ? p.k : p.q;
    float dw[16] = {};
    f32x8 w1 = {}, w2 = {};
    if (mine && j0 < half) {
        w1 = weight8(p, x.weight, j0);
        w2 = weight8(p, x.weight, half + j0);
    }
    for (int64_t t0 = (int64_t)w.line * TOK; mine && t0 < p.total_len; t0 += (int64_t)a.lines * TOK) {
        const bool row = t0 + sub < p.total_len, on = row && j0 < half;
        const int t = row ? (int)t0 + sub : 0;
        const T* in = (const T*)x.x + (int64_t)t * x.st + j0;
        const T* din = (const T*)x.d + (int64_t)t * x.d_st + j0;
        T* out = (T*)x.y + (int64_t)t * x.y_st + j0;
        vec8 a1 = {}, a2 = {}, d1 = {}, d2 = {};
        auto load = [&](int h, vec8& v1, vec8& v2, vec8& e1, vec8& e2) {
            v1 = *(const vec8*)(in + (int64_t)h * x.sh);
            v2 = *(const vec8*)(in + (int64_t)h * x.sh + half);
            e1 = *(const vec8*)(din + (int64_t)h * x.d_sh);
            e2 = *(const vec8*)(din + (int64_t)h * x.d_sh + half);
        };
        if (on) load(w.first, a1, a2, d1, d2);
        const int pos = row ? position(p, t) : -1;
        const bool has = on && pos >= 0;
        f32x8 c1 = {}, c2 = {}, s1 = {}, s2 = {};
        if (has) {
            const int64_t at = (int64_t)pos * p.head_dim + j0;
            c1 = *(const f32x8*)(p.cos + at);
            c2 = *(const f32x8*)(p.cos + at + half);
            s1 = *(const f32x8*)(p.sin + at);
            s2 = *(const f32x8*)(p.sin + at + half);
        } else {  // (whatever a row without a position holds counts as zeros)
            a1 = a2 = d1 = d2 = vec8{};
        }
        for (int h = w.first; h < w.last; ++h) {
            vec8 n1 = {}, n2 = {}, g1 = {}, g2 = {};
            if (has && h + 1 < w.last) load(h + 1, n1, n2, g1, g2);
            float f1[8], f2[8], dn1[8], dn2[8], ss = 0.f, sd = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f1[e] = to_float(a1[e]);
                f2[e] = to_float(a2[e]);
                const float u1 = to_float(d1[e]), u2 = to_float(d2[e]);
                dn1[e] = u1 * c1[e] + u2 * s2[e];
                dn2[e] = u2 * c2[e] - u1 * s1[e];
                ss += f1[e] * f1[e] + f2[e] * f2[e];
                sd += dn1[e] * w1[e] * f1[e] + dn2[e] * w2[e] * f2[e];
            }
            ss = sum_lanes<LP>(ss);
            sd = sum_lanes<LP>(sd);
            // (lanes without a row add nothing to the weights' gradients, whatever eps)
            const float r = has ? 1.f / sqrtf(ss * inv_d + p.eps) : 0.f, k = r * r * (sd * inv_d);
            vec8 o1, o2;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[e] += dn1[e] * (f1[e] * r);
                dw[8 + e] += dn2[e] * (f2[e] * r);
                o1[e] = from_float<T>(r * (dn1[e] * w1[e] - f1[e] * k));
                o2[e] = from_float<T>(r * (dn2[e] * w2[e] - f2[e] * k));
            }
            if (on) {  // (zeros where there is no position)
                *(vec8*)(out + (int64_t)h * x.y_sh) = o1;
                *(vec8*)(out + (int64_t)h * x.y_sh + half) = o2;
            }
            a1 = n1;
            a2 = n2;
            d1 = g1;
            d2 = g2;
        }
    }
    // the block's part of the weights' gradients
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float v = dw[e];
#pragma unroll
        for (int o = LP; o < 64; o <<= 1) v += wave_xor(v, o);
        if (sub == 0) sums[wv][part * 16 + e] = v;
    }
    if (lane == 0) side_of[wv] = mine ? w.side : 2;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += kThreads) {
        const int side = i >= p.head_dim, d = i - side * p.head_dim, second = d >= half, j = d - second * half;
        const int at = (j / 8) * 16 + second * 8 + j % 8;
        float v = 0.f;
#pragma unroll
        for (int n = 0; n < kWaves; ++n) v += side_of[n] == side ? sums[n][at] : 0.f;
        p.ws[(int64_t)blockIdx.x * 2 * p.head_dim + i] = v;
    }
}

// The blocks' parts joined: a block takes 16 elements, 64 threads each.
__global__ __launch_bounds__(1024) void qk_norm_rope_join_kernel(QkNormParams p, int parts) {
    __shared__ float sums[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, i = blockIdx.x * 16 + c, n = 2 * p.head_dim;
    float v = 0.f;
    int b = r;
    for (; b + 7 * 64 < parts; b += 8 * 64) {  // eight requests on their way at a time
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = p.ws[(int64_t)(b + e * 64) * n + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) v += u[e];
    }
    for (; b < parts; b += 64) v += p.ws[(int64_t)b * n + i];
    sums[r][c] = v;
    for (int o = 32; o >= 1; o >>= 1) {
        __syncthreads();
        if (r < o) sums[r][c] += sums[r + o][c];
    }
    if (r == 0) {
        float* dw = i < p.head_dim ? p.q.dw : p.k.dw;
        if (dw) dw[i < p.head_dim ? i : i - p.head_dim] = sums[0][c];
    }
}

int lanes_of(int head_dim) {
    int n = 1;
    while (n * 16 < head_dim) n <<= 1;
    return n;
}

// As many waves as are resident at once (the backward pass has registers for twelve a unit, eight in float32, the forward for
// sixteen), each with every so many-th group of tokens, and up to four heads to a wave where that leaves enough waves: a token's
// cosines are read once for them.  32768 tokens, 16 and 2 heads of 128, bfloat16, us: forward 70.5 (two heads 71.8, eight 73.3;
// 2048 waves 86, 8192 waves 69.8, and then 9.1 instead of 7.4 at 2049 tokens), backward 100.3 (eight heads 99.6, sixteen 106.7;
// 1536 waves 120, 6144 waves 103); 16001 tokens, 16 and 16 heads of 64, backward, a call
// among others, 47 (sixteen heads 47, 6144 waves 48; with queries and keys in every wave's turn, which needs 224 registers, 61).
// The float16 backward keeps two registers of a lane in memory for heads of 32 to 64 and past 128.
QkPlan qk_plan(int total_len, int q_heads, int k_heads, int head_dim, int most) {
    const int tok = 64 / lanes_of(head_dim);
    const int64_t groups = ((int64_t)total_len + tok - 1) / tok;
    int n = 1;
    auto chunks = [&](int heads) { return heads / n + (heads % n != 0); };
    while (n < 4 && groups * ((int64_t)chunks(q_heads) + chunks(k_heads)) > most) n *= 2;
    QkPlan a;
    a.q_chunks = chunks(q_heads);
    a.chunks = a.q_chunks + chunks(k_heads);
    a.q_heads = a.q_chunks ? (q_heads - 1) / a.q_chunks + 1 : 0;
    a.k_heads = a.chunks > a.q_chunks ? (k_heads - 1) / (a.chunks - a.q_chunks) + 1 : 0;
    a.lines = a.chunks ? (int)std::min(groups, (int64_t)std::max(1, most / a.chunks)) : 0;  // (no heads: no blocks)
    a.blocks = (int)(((int64_t)a.lines * a.chunks + kWaves - 1) / kWaves);
    return a;
}

int bwd_waves(int dtype) { return 256 * (dtype == 0 ? 8 : 12); }

template <typename T, int LP>
hipError_t run(const QkNormParams& p, const QkPlan& a, bool backward, hipStream_t stream) {
    if (backward) DSALT_LAUNCH("qk_norm_rope_bwd", (qk_norm_rope_bwd_kernel<T, LP>), dim3(a.blocks), dim3(kThreads), 0, stream, p, a);
    else DSALT_LAUNCH("qk_norm_rope", (qk_norm_rope_kernel<T, LP>), dim3(a.blocks), dim3(kThreads), 0, stream, p, a);
    return hipGetLastError();
}

template <typename T>
hipError_t run_lanes(const QkNormParams& p, const QkPlan& a, bool backward, hipStream_t stream) {
    switch (lanes_of(p.head_dim)) {
        case 1: return run<T, 1>(p, a, backward, stream);
        case 2: return run<T, 2>(p, a, backward, stream);
        case 4: return run<T, 4>(p, a, backward, stream);
        case 8: return run<T, 8>(p, a, backward, stream);
        default: return run<T, 16>(p, a, backward, stream);
    }
}

hipError_t run_type(const QkNormParams& p, const QkPlan& a, bool backward, hipStream_t stream) {
    switch (p.dtype) {
        case 0: return run_lanes<float>(p, a, backward, stream);
        case 1: return run_lanes<bf16>(p, a, backward, stream);
        default: return run_lanes<f16>(p, a, backward, stream);
    }
}

}  // namespace

hipError_t qk_norm_rope_launch(const QkNormParams& p, hipStream_t stream) {
    if (p.total_len == 0 || p.q.heads + p.k.heads == 0) return hipSuccess;
    return run_type(p, qk_plan(p.total_len, p.q.heads, p.k.heads, p.head_dim, 256 * 16), false, stream);
}

size_t qk_norm_rope_bwd_ws_bytes(int total_len, int q_heads, int k_heads, int head_dim, int dtype) {
    return (size_t)qk_plan(total_len, q_heads, k_heads, head_dim, bwd_waves(dtype)).blocks * 2 * head_dim * sizeof(float);
}

// (a batch without rows: the join alone, which writes zeros)
hipError_t qk_norm_rope_bwd_launch(const QkNormParams& p, hipStream_t stream) {
    if (p.q.heads + p.k.heads == 0) return hipSuccess;
    const QkPlan a = qk_plan(p.total_len, p.q.heads, p.k.heads, p.head_dim, bwd_waves(p.dtype));
    if (a.blocks > 0)
        if (hipError_t e = run_type(p, a, true, stream)) return e;
    DSALT_LAUNCH("qk_norm_rope_join", qk_norm_rope_join_kernel, dim3(p.head_dim / 8), dim3(1024), 0, stream, p, a.blocks);
    return hipGetLastError();
}

}  // namespace dsalt
