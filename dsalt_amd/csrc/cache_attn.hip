// Attention of query tokens over the paged 8-bit cache: row t is the token at position pos[t] of request
// req[t] and attends A(i) = [i - w + 1, i] U {landmarks p of its head's set : 0 <= p < i - w + 1}.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j + b_j - m): one pass with a running maximum m and
// sum.  What bounds it is the cache: 2 D bytes a key for two products of D each.  A row's query heads of one
// key/value head attend the same window, so a block takes a row, a key/value head and up to 16 of its query
// heads, and forms both products of the window on the matrix cores; landmarks are a head's own and are taken a
// wave a head with ordinary arithmetic.  Both keep 32-bit scores, weights and sums.
#include "cache.h"
#include "common.h"
#include "fp8.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kStep = 32;  // window keys a wave takes at a time
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

// number of bfloat16 parts of a query element (exact: 8, 11 and 24 bits) and of a weight (16 bits of it for
// 16-bit outputs, 24 for float32)
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int q = 1, p = 2; };
template <> struct Parts<f16> { static constexpr int q = 2, p = 2; };
template <> struct Parts<float> { static constexpr int q = 3, p = 3; };

struct AttnPlan {
    int ns;      // splits of a row's window
    int nl;      // splits that take landmarks
    int tiles;   // blocks of up to 16 query heads of a key/value head
    int nh;      // heads of a block (the last one may hold fewer)
    int chunks;  // parts of a head's landmark slots within a block
};

__device__ __forceinline__ uint32_t half_pair(uint32_t a, uint32_t b, bool hi) {  // halves of a and b side by side
    return __builtin_amdgcn_perm(b, a, hi ? 0x07060302u : 0x05040100u);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32: to 1 ulp, 0 below 2^-126

// eight elements of a 16-byte aligned row as floats
template <typename T>
__device__ __forceinline__ void load8(const T* x, float* f) {
    typedef T vec __attribute__((ext_vector_type(8), aligned(16)));
    const vec v = *(const vec*)x;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_float(v[e]);
}

// eight floats into PARTS bfloat16 operands that sum to them
template <int PARTS>
__device__ __forceinline__ void split8(const float* x, bf16x8* o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float r = x[e];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
            const bf16 h = (bf16)r;
            o[k][e] = h;
            r -= (float)h;
        }
    }
}

// Parts of a block's result: the waves' shares of the window, then the chunks of the landmarks.
// ml: running maximum (of logits in base 2) and sum of each part and head; acc: its weighted sum of values.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void cache_attn_kernel(CacheAttnParams p, AttnPlan a) {
    constexpr int QP = Parts<T>::q, PP = Parts<T>::p, KS = D / 32, JN = D / 16, DL = D / 4;
    extern __shared__ float lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, row16 = lane & 15, kg = lane >> 4;
    const int G = p.c.n_kv, group = p.n_heads / G, bt_log = p.c.bt_log, bt = 1 << bt_log;
    const int hx = blockIdx.x % a.tiles, tg = blockIdx.x / a.tiles, g = tg % G, t = tg / G, split = blockIdx.y;
    const int h0 = g * group + hx * 16, nh = min(16, group - hx * 16);
    const int parts = kWaves + a.chunks;
    float2* ml = (float2*)lds;
    float* accs = lds + 2 * parts * a.nh;
    const int req = p.req[t], pos = p.pos[t];
    const bool live = req >= 0 && req < p.n_reqs && pos >= 0;
    const int low = live ? max(pos - max(p.w[t], 1) + 1, 0) : 0;
    const int32_t* table = p.table + (live ? (int64_t)req * p.table_st : 0);
    const float scale2 = p.scale * kLog2e;

    // ---- window: keys base + 32 step ..., from the aligned position at or before the first
    {
        const int base = low & ~(kStep - 1);
        const int end = min(pos, (p.cols << bt_log) - 1);  // what the table can name
        const int steps = live && end >= low ? ((end - base) >> 5) + 1 : 0, per = ceil_div(steps, a.ns);
        const int s0 = split * per, s1 = min(steps, s0 + per);
        // q: lane (head row16, kg) holds elements kg D/4 + 8 s + e
        bf16x8 qf[KS][QP];
        {
            const T* qr = (const T*)p.q + (int64_t)t * p.q_st + (int64_t)(h0 + min(row16, nh - 1)) * p.q_sh + kg * DL;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                float x[8];
                load8(qr + 8 * s, x);
                split8<QP>(x, qf[s]);
            }
        }
        floatx4 acc[JN];
#pragma unroll
        for (int j = 0; j < JN; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        const int first = s0 + wv, mine = first < s1 ? (s1 - 1 - first) / kWaves + 1 : 0;
        for (int b0 = 0; b0 < mine; b0 += 32) {
            // lane 2 i + half: page and scales of the 16 keys `half` of step i of this batch
            const int pk = base + (first + (b0 + (lane >> 1)) * kWaves) * kStep + (lane & 1) * 16;
            int page = -1;
            float ks = 0.f, vs = 0.f;
            if (b0 + (lane >> 1) < mine && (pk >> bt_log) < p.cols) {
                page = table[pk >> bt_log];
                if (page < 0 || page >= p.c.n_blocks) page = -1;
                else {
                    ks = p.c.ks[(int64_t)page * G + g];
                    vs = p.c.vs[(int64_t)page * G + g];
                }
            }
            const int n = min(32, mine - b0);
            u32x4 kr[2][DL / 16];
            typedef uint32_t vword __attribute__((ext_vector_type(JN / 4)));
            vword vr[8];
            auto tile_at = [&](int i, int half) -> int64_t {  // bytes before the 16 keys (page 0 where there is none)
                const int pg = max(__builtin_amdgcn_readlane(page, 2 * i + half), 0);
                const int at = base + (first + (b0 + i) * kWaves) * kStep + half * 16;
                return ((((int64_t)pg * G + g) << bt_log) + (at & (bt - 1))) * D;
            };
            auto load_k = [&](int i) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint8_t* x = p.c.k + tile_at(i, half) + row16 * D + kg * DL;
#pragma unroll
                    for (int c = 0; c < DL / 16; ++c) kr[half][c] = *(const u32x4*)(x + 16 * c);
                }
            };
            auto load_v = [&](int i) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint8_t* x = p.c.v + tile_at(i, half) + (4 * kg) * D + row16 * JN;
#pragma unroll
                    for (int e = 0; e < 4; ++e) vr[4 * half + e] = *(const vword*)(x + e * D);
                }
            };
            load_k(0);
            load_v(0);
            for (int i = 0; i < n; ++i) {
                const int at = base + (first + (b0 + i) * kWaves) * kStep;
                const int pg0 = __builtin_amdgcn_readlane(page, 2 * i), pg1 = __builtin_amdgcn_readlane(page, 2 * i + 1);
                auto scale_lane = [&](float x, int half) {
                    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 2 * i + half));
                };
                // scores of keys at + 16 half + 4 kg + r for head row16
                floatx4 sc[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    sc[half] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        uint32_t f[4];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t u = kr[half][s / 2][(s & 1) * 2 + e];
                            f[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.f, false));
                            f[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.f, true));
                        }
                        const bf16x8 kf = __builtin_bit_cast(bf16x8, u32x4{f[0], f[1], f[2], f[3]});
#pragma unroll
                        for (int k = 0; k < QP; ++k) sc[half] = mma(kf, qf[s][k], sc[half]);
                    }
                }
                if (i + 1 < n) load_k(i + 1);
                const bool whole = at >= low && at + kStep - 1 <= end && pg0 >= 0 && pg1 >= 0;
                float x[8];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float f = scale_lane(ks, half) * scale2;
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[4 * half + r] = sc[half][r] * f;
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int j = at + (e & 4) * 4 + 4 * kg + (e & 3);
                        if (j < low || j > end || (e < 4 ? pg0 : pg1) < 0) {
                            x[e] = -INFINITY;
                            vr[e] = vword{};
                        }
                    }
                }
                float mx = x[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
                mx = max_g4(mx);
                if (__any(mx > m)) {
                    const float m1 = fmaxf(m, mx), f = m == -INFINITY ? 0.f : exp2_(m - m1);
                    m = m1;
                    l *= f;
#pragma unroll
                    for (int j = 0; j < JN; ++j) acc[j] *= f;
                }
                const float mb = m == -INFINITY ? 0.f : m;
                const float v0 = scale_lane(vs, 0), v1 = scale_lane(vs, 1);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = exp2_(x[e] - mb);
                    l += w;
                    x[e] = w == 0.f ? 0.f : w * (e < 4 ? v0 : v1);  // (a scale behind masked keys may be anything)
                }
                bf16x8 pf[PP];
                split8<PP>(x, pf);
                // values: the lane's word of key e holds elements JN row16 ...; operand j takes byte j of all eight
#pragma unroll
                for (int j = 0; j < JN; j += 2) {
                    uint32_t c[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t u = vr[e][j / 4];
                        c[e] = (j & 2) ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.f, true))
                                       : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.f, false));
                    }
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const bf16x8 vf = __builtin_bit_cast(
                            bf16x8, u32x4{half_pair(c[0], c[1], hi), half_pair(c[2], c[3], hi), half_pair(c[4], c[5], hi),
                                          half_pair(c[6], c[7], hi)});
#pragma unroll
                        for (int k = 0; k < PP; ++k) acc[j + hi] = mma(vf, pf[k], acc[j + hi]);
                    }
                }
                if (i + 1 < n) load_v(i + 1);
            }
        }
        l = sum_g4(l);
        if (row16 < nh) {
            if (kg == 0) ml[wv * a.nh + row16] = make_float2(m, l);
            if (mine > 0) {
                float* o = accs + (wv * a.nh + row16) * D + kg * DL;  // element JN r + j of the lane's quarter
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < JN; ++j) o[r * JN + j] = acc[j][r];
            }
        }
    }

    // ---- landmarks: D / 16 lanes a key, 16 elements each; every group of lanes keeps its own running maximum
    const bool marks = split < a.nl;
    if (marks) {
        constexpr int LPK = D / 16, KPW = 64 / LPK;
        const int part = lane % LPK, sub = lane / LPK;
        const int kl = ceil_div(p.k_lmk, a.nl), k0 = min(split * kl, p.k_lmk), k1 = min(k0 + kl, p.k_lmk);
        const int kc = ceil_div(k1 - k0, a.chunks);
        for (int it = wv; it < nh * a.chunks; it += kWaves) {
            const int hh = it / a.chunks, c = it - hh * a.chunks, h = h0 + hh;
            const int c0 = min(k0 + c * kc, k1), c1 = live ? min(c0 + kc, k1) : c0;
            const int64_t set = live ? ((int64_t)h * p.n_reqs + req) * p.k_lmk : 0;
            const T* qr = (const T*)p.q + (int64_t)t * p.q_st + (int64_t)h * p.q_sh + part * 16;
            float q[16], acc[16], m = -INFINITY, l = 0.f;
            load8(qr, q);
            load8(qr + 8, q + 8);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                q[e] *= scale2;
                acc[e] = 0.f;
            }
            for (int b = c0; b < c1; b += 64) {
                // lane: one slot's place in the cache, scales and bias
                int64_t off = -1;
                float ks = 0.f, vs = 0.f, bias = 0.f;
                if (b + lane < c1) {
                    const int j = p.lmk[set + b + lane];
                    const int bl = j >> bt_log;
                    const int page = j >= 0 && j < low && bl < p.cols ? table[bl] : -1;
                    if (page >= 0 && page < p.c.n_blocks) {
                        const int64_t tile = (int64_t)page * G + g;
                        off = ((tile << bt_log) + (j & (bt - 1))) * D;
                        ks = p.c.ks[tile];
                        vs = p.c.vs[tile];
                        if (p.lbias) bias = p.lbias[set + b + lane] * kLog2e;
                    }
                }
                const int n = min(64, c1 - b);
                for (int i = 0; i < n; i += KPW) {
                    const int64_t at = __shfl(off, i + sub);
                    const bool on = at >= 0;
                    if (!__any(on)) continue;
                    u32x4 ku = {}, vu = {};
                    if (on) {
                        ku = *(const u32x4*)(p.c.k + at + part * 16);
                        vu = *(const u32x4*)(p.c.v + at + part * 16);
                    }
                    float f[16], s = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) e4m3_x4(ku[e], f + 4 * e);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s += q[e] * f[e];
#pragma unroll
                    for (int o = 1; o < LPK; o <<= 1) s += wave_xor(s, o);
                    const float kss = __shfl(ks, i + sub), vss = __shfl(vs, i + sub), bs = __shfl(bias, i + sub);
                    s = on ? s * kss + bs : -INFINITY;
                    const float m1 = fmaxf(m, s), mb = m1 == -INFINITY ? 0.f : m1;
                    const float fa = exp2_(m - mb), pr = on ? exp2_(s - mb) : 0.f;
                    l = l * fa + pr;
#pragma unroll
                    for (int e = 0; e < 4; ++e) e4m3_x4(vu[e], f + 4 * e);
                    const float pv = pr * vss;
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[e] = acc[e] * fa + pv * f[e];
                    m = m1;
                }
            }
            float mw = m;
#pragma unroll
            for (int o = LPK; o < 64; o <<= 1) mw = fmaxf(mw, wave_xor(mw, o));
            const float fa = mw == -INFINITY ? 1.f : exp2_(m - mw);
            l *= fa;
#pragma unroll
            for (int o = LPK; o < 64; o <<= 1) l += wave_xor(l, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[e] *= fa;
#pragma unroll
                for (int o = LPK; o < 64; o <<= 1) acc[e] += wave_xor(acc[e], o);
            }
            const int slot = (kWaves + c) * a.nh + hh;
            if (lane == 0) ml[slot] = make_float2(mw, l);
            if (sub == 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) accs[slot * D + part * 16 + e] = acc[e];
            }
        }
    }
    __syncthreads();

    // ---- the parts joined
    const int np = marks ? parts : kWaves;
    for (int i = tid; i < nh * D; i += kThreads) {
        const int hh = i / D, d = i - hh * D;
        float M = -INFINITY, L = 0.f, o = 0.f;
        for (int k = 0; k < np; ++k) M = fmaxf(M, ml[k * a.nh + hh].x);
        const float mb = M == -INFINITY ? 0.f : M;
        for (int k = 0; k < np; ++k) {
            const float2 v = ml[k * a.nh + hh];
            if (v.y == 0.f) continue;  // nothing attended there
            const float f = v.x == -INFINITY ? 1.f : exp2_(v.x - mb);
            L += v.y * f;
            o += accs[(k * a.nh + hh) * D + d] * f;
        }
        const int64_t th = (int64_t)t * p.n_heads + h0 + hh;
        if (a.ns > 1) {
            const int64_t at = th * a.ns + split;
            if (d == 0) ((float2*)p.ws)[at] = make_float2(M, L);
            if (L != 0.f) ((float*)p.ws)[2 * (int64_t)p.n_rows * p.n_heads * a.ns + at * D + d] = o;
        } else {
            ((T*)p.out)[(int64_t)t * p.o_st + (int64_t)(h0 + hh) * p.o_sh + d] = from_float<T>(L == 0.f ? 0.f : o / L);
            if (d == 0) p.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        }
    }
}

// The splits of a row and head joined: a block of D threads each.
template <typename T, int D>
__global__ __launch_bounds__(D) void cache_attn_join_kernel(CacheAttnParams p, int ns) {
    const int64_t th = blockIdx.x;
    const int t = (int)(th / p.n_heads), h = (int)(th - (int64_t)t * p.n_heads), d = threadIdx.x;
    const float2* ml = (const float2*)p.ws + th * ns;
    const float* acc = (const float*)p.ws + 2 * (int64_t)p.n_rows * p.n_heads * ns + th * ns * D + d;
    float M = -INFINITY, L = 0.f, o = 0.f;
    for (int k = 0; k < ns; ++k) M = fmaxf(M, ml[k].x);
    const float mb = M == -INFINITY ? 0.f : M;
    for (int k = 0; k < ns; ++k) {
        const float2 v = ml[k];
        if (v.y == 0.f) continue;
        const float f = v.x == -INFINITY ? 1.f : exp2_(v.x - mb);
        L += v.y * f;
        o += acc[(int64_t)k * D] * f;
    }
    ((T*)p.out)[(int64_t)t * p.o_st + (int64_t)h * p.o_sh + d] = from_float<T>(L == 0.f ? 0.f : o / L);
    if (d == 0) p.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

AttnPlan attn_plan(const CacheAttnParams& p) {
    AttnPlan a;
    const int group = p.n_heads / p.c.n_kv;
    a.tiles = ceil_div(group, 16);
    a.nh = group < 16 ? group : 16;
    a.chunks = p.k_lmk == 0 ? 0 : a.nh < kWaves ? kWaves / a.nh : 1;
    // splits: about four blocks a CU, none of less than four steps a wave
    const int64_t cap = (int64_t)p.cols << p.c.bt_log;
    const int64_t w = p.w_max > 0 && p.w_max < cap ? p.w_max : cap;
    const int64_t blocks = (int64_t)p.n_rows * p.c.n_kv * a.tiles, most = (w / kStep + 1) / (4 * kWaves);
    int64_t ns = (1024 + blocks - 1) / blocks;
    ns = ns < most ? ns : most;
    a.ns = (int)(ns < 1 ? 1 : ns);
    const int nl = ceil_div(p.k_lmk, 64);
    a.nl = nl < a.ns ? nl : a.ns;
    return a;
}

}  // namespace

size_t cache_attn_ws_bytes(const CacheAttnParams& p) {
    const AttnPlan a = attn_plan(p);
    return a.ns > 1 ? (size_t)p.n_rows * p.n_heads * a.ns * (p.c.head_dim + 2) * sizeof(float) : 0;
}

hipError_t cache_attn_launch(const CacheAttnParams& p, hipStream_t stream) {
    if (p.n_rows == 0) return hipSuccess;
    const AttnPlan a = attn_plan(p);
    const dim3 grid((unsigned)((int64_t)p.n_rows * p.c.n_kv * a.tiles), (unsigned)a.ns);
    const unsigned lds = (unsigned)((kWaves + a.chunks) * a.nh * (p.c.head_dim + 2) * sizeof(float));
    const dim3 join((unsigned)((int64_t)p.n_rows * p.n_heads));
#define RUN(T, DD)                                                                                                        \
    do {                                                                                                                  \
        if (lds > 65536)                                                                                                  \
            if (hipError_t e = hipFuncSetAttribute((const void*)cache_attn_kernel<T, DD>,                                 \
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024))               \
                return e;                                                                                                 \
        DSALT_LAUNCH("cache_attn", (cache_attn_kernel<T, DD>), grid, dim3(kThreads), lds, stream, p, a);                  \
        if (a.ns > 1) DSALT_LAUNCH("cache_attn_join", (cache_attn_join_kernel<T, DD>), join, dim3(DD), 0, stream, p, a.ns); \
    } while (0)
    const bool wide = p.c.head_dim == 128;
    switch (p.dtype) {
        case 0:
            if (wide) RUN(float, 128);
            else RUN(float, 64);
            break;
        case 1:
            if (wide) RUN(bf16, 128);
            else RUN(bf16, 64);
            break;
        default:
            if (wide) RUN(f16, 128);
            else RUN(f16, 64);
            break;
    }
#undef RUN
    return hipGetLastError();
}

}  // namespace dsalt
