// Attention of query tokens over the paged 8-bit cache: row t is the token at position pos[t] of request
// req[t] and attends A(i) = [i - w + 1, i] U {landmarks p of its head's set : 0 <= p < i - w + 1}.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j + b_j - m): one pass with a running maximum m and
// sum.  What bounds it is the cache: 2 D bytes a key for two products of D each.  A row's query heads of one
// key/value head attend the same window, so a block takes a row, a key/value head and up to 16 of its query
// heads, and forms both products of the window on the matrix cores; landmarks are a head's own and are taken a
// wave a head with ordinary arithmetic.  Both keep 32-bit scores, weights and sums.
#include <algorithm>

#include "cache.h"
#include "common.h"
#include "fp8.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kStep = 32;  // window keys a wave takes at a time
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

// number of bfloat16 parts of a query element (exact: 8, 11 and 24 bits) and of a weight: 16 bits of it for
// 16-bit outputs, whose own rounding, half a step of 2^-8 or 2^-11 of a value, is far coarser, 24 for float32 (lists keep
// weights in float32)
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int q = 1, p = 2; };
template <> struct Parts<f16> { static constexpr int q = 2, p = 2; };
template <> struct Parts<float> { static constexpr int q = 3, p = 3; };

// waves a SIMD that the registers are held to (168, 128 and 256 of them)
template <typename T, int D> struct MinWaves { static constexpr int value = D == 64 ? 4 : 3; };
template <> struct MinWaves<float, 64> { static constexpr int value = 3; };
template <> struct MinWaves<float, 128> { static constexpr int value = 2; };

struct AttnPlan {
    bool list;   // a block a row and head; otherwise a row and a key/value head
    int ns;      // splits of a row's window
    int nl;      // splits that take landmarks (groups)
    int tiles;   // blocks of a key/value head's query heads
    int nh;      // heads of a block (the last one may hold fewer)
    int waves;   // of a block
    int chunks;  // parts of a head's landmark slots within a block (groups)
};

__device__ __forceinline__ uint32_t half_pair(uint32_t a, uint32_t b, bool hi) {  // halves of a and b side by side
    return __builtin_amdgcn_perm(b, a, hi ? 0x07060302u : 0x05040100u);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32: to 1 ulp, 0 below 2^-126

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
// sum over the N = 4 or 8 lanes that share lane / N (every one gets it)
template <int N>
__device__ __forceinline__ float sum_in(float v) {
    v += dpp<0xb1>(v);  // lanes 1, 0, 3, 2 of each four
    v += dpp<0x4e>(v);  // 2, 3, 0, 1
    return N == 8 ? v + dpp<0x141>(v) : v;  // the other four of each eight
}
// sum and maximum over the 64 / N lanes that share lane mod N
template <int N>
__device__ __forceinline__ float sum_over(float v) {
    if (N == 4) v += dpp<0x124>(v);  // four lanes on within each sixteen
    return sum_g4(v + dpp<0x128>(v));
}
template <int N>
__device__ __forceinline__ float max_over(float v) {
    if (N == 4) v = fmaxf(v, dpp<0x124>(v));
    return max_g4(fmaxf(v, dpp<0x128>(v)));
}

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

// One query row: its request's table, the first position of its window and the last that the table can name.
struct Row {
    int req, low, end;
    bool live;
    const int32_t* table;
    __device__ __forceinline__ Row(const CacheAttnParams& p, int t) {
        req = p.req[t];
        const int pos = p.pos[t];
        live = req >= 0 && req < p.n_reqs && pos >= 0;
        low = live ? max(pos - max(p.w[t], 1) + 1, 0) : 0;
        end = live ? min(pos, (p.cols << p.c.bt_log) - 1) : -1;
        table = p.table + (live ? (int64_t)req * p.table_st : 0);
    }
};

constexpr uint32_t kNone = 0xffffffffu;

struct Slot {      // a key in the cache: page, head and token in one number (fewer than 2^32 - 1), kNone: not attended;
    uint32_t key;  // its scales and bias, not looked at for kNone
    float ks, vs, bias;
};

// Keys of one head taken from a list: D / 16 lanes a key, 16 elements each.  A wave takes NB at a time, a lane
// having looked one up; every group of lanes keeps its own maximum, sum and output, joined at the end.
template <typename T, int D, int NS_>
struct List {
    static constexpr int LPK = D / 16, KPW = 64 / LPK, NS = NS_, NB = NS * KPW;
    const CacheAttnParams& p;
    const Row& r;
    int g, part, sub;
    float q[16], acc[16], m, l;

    __device__ __forceinline__ List(const CacheAttnParams& p_, const Row& r_, int g_) : p(p_), r(r_), g(g_) {
        const int lane = threadIdx.x & 63;
        part = lane % LPK;
        sub = lane / LPK;
    }
    __device__ __forceinline__ void begin(const T* head) {
        load8(head + part * 16, q);
        load8(head + part * 16 + 8, q + 8);
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            q[e] *= p.scale * kLog2e;
            acc[e] = 0.f;
        }
    }
    // a bias in base 2 (the type's lowest values stay finite, as masks of them are apart from minus infinity)
    __device__ __forceinline__ static float base2(float b) { return b > -INFINITY ? fmaxf(b * kLog2e, -3e38f) : b; }
    // the page of position j where it is attended, else -1
    __device__ __forceinline__ int page(int j, bool attended) const {
        const int b = j >> p.c.bt_log;
        const bool in = attended && j >= 0 && b < p.cols;
        const int pg = r.table[in ? b : 0];
        return in && pg >= 0 && pg < p.c.n_blocks ? pg : -1;
    }
    // (a bias of minus infinity masks its key, so that what the cache holds there is not read)
    __device__ __forceinline__ Slot place(int j, int pg, int64_t bias_at) const {
        const uint32_t tile = (uint32_t)max(pg, 0) * (uint32_t)p.c.n_kv + (uint32_t)g;
        const uint32_t key = (tile << p.c.bt_log) + (uint32_t)(j & ((1 << p.c.bt_log) - 1));
        const float bias = p.lbias && bias_at >= 0 ? p.lbias[bias_at] : 0.f;
        return Slot{pg < 0 || bias == -INFINITY ? kNone : key, p.c.ks[tile], p.c.vs[tile], bias};
    }
    // the wave's NB slots (`n` of them used); `next` is called once the batch's keys and values are requested
    template <typename F>
    __device__ __forceinline__ void take(const Slot& s, int n, F next) {
        const int used = ceil_div(n, KPW);
        u32x4 ku[NS], vu[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i >= used) break;
            const uint32_t key = __shfl(s.key, i * KPW + sub);
            ku[i] = vu[i] = u32x4{};
            if (key != kNone) {
                ku[i] = *(const u32x4*)(p.c.k + (uint64_t)key * D + part * 16);
                vu[i] = *(const u32x4*)(p.c.v + (uint64_t)key * D + part * 16);
            }
        }
        next();
        float x[NS], f[16], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            x[i] = -INFINITY;
            if (i >= used) continue;
            const bool on = __shfl(s.key, i * KPW + sub) != kNone;
            const float ks = __shfl(s.ks, i * KPW + sub), bias = p.lbias ? base2(__shfl(s.bias, i * KPW + sub)) : 0.f;
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) e4m3_x4(ku[i][e], f + 4 * e);
#pragma unroll
            for (int e = 0; e < 16; ++e) d += q[e] * f[e];
            d = sum_in<LPK>(d);
            if (on) x[i] = d * ks + bias;
            mx = fmaxf(mx, x[i]);
        }
        const float m1 = fmaxf(m, mx), mb = m1 == -INFINITY ? 0.f : m1, fa = exp2_(m - mb);
        m = m1;
        l *= fa;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] *= fa;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (i >= used) break;
            const float vs = __shfl(s.vs, i * KPW + sub);
            const float pr = exp2_(x[i] - mb), pv = pr == 0.f ? 0.f : pr * vs;
            l += pr;
#pragma unroll
            for (int e = 0; e < 4; ++e) e4m3_x4(vu[i][e], f + 4 * e);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[e] += pv * f[e];
        }
    }
    // the wave's result: (maximum, sum) and the weighted sum of values [D]
    __device__ __forceinline__ void end(float2* ml, float* out) {
        const float mw = max_over<LPK>(m), fa = mw == -INFINITY ? 1.f : exp2_(m - mw);
        l = sum_over<LPK>(l * fa);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = sum_over<LPK>(acc[e] * fa);
        if ((threadIdx.x & 63) == 0) *ml = make_float2(mw, l);
        if (sub == 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) out[part * 16 + e] = acc[e];
        }
    }
};

// A block's parts joined, `np` for each of its nh heads (ml and accs [part][stride heads]): written out, or to the
// workspace where the row is split.  A part with sum 0 attended nothing and left no values.
template <typename T, int D, int THREADS>
__device__ void join_parts(const CacheAttnParams& p, float2* ml, const float* accs, int np, int stride, int nh, int t, int h0, int split,
                           int ns) {
    float2* total = ml + np * stride;  // maximum and sum of each head
    __syncthreads();
    for (int hh = threadIdx.x; hh < nh; hh += THREADS) {
        float M = -INFINITY, L = 0.f;
        for (int k = 0; k < np; ++k) M = fmaxf(M, ml[k * stride + hh].x);
        const float mb = M == -INFINITY ? 0.f : M;
        for (int k = 0; k < np; ++k) {
            const float2 v = ml[k * stride + hh];
            const float f = v.x == -INFINITY ? 1.f : exp2_(v.x - mb);
            if (v.y != 0.f) L += v.y * f;
            ml[k * stride + hh].x = f;
        }
        total[hh] = make_float2(M, L);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * D; i += THREADS) {
        const int hh = i / D, d = i - hh * D;
        float o = 0.f;
        for (int k = 0; k < np; ++k) {
            const float2 v = ml[k * stride + hh];
            if (v.y != 0.f) o += accs[(k * stride + hh) * D + d] * v.x;
        }
        const float M = total[hh].x, L = total[hh].y;
        const int64_t th = (int64_t)t * p.n_heads + h0 + hh;
        if (ns > 1) {
            const int64_t at = th * ns + split;
            if (d == 0) ((float2*)p.ws)[at] = make_float2(M, L);
            if (L != 0.f) ((float*)p.ws)[2 * (int64_t)p.n_rows * p.n_heads * ns + at * D + d] = o;
        } else {
            ((T*)p.out)[(int64_t)t * p.o_st + (int64_t)(h0 + hh) * p.o_sh + d] = from_float<T>(L == 0.f ? 0.f : o / L);
            if (d == 0) p.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        }
    }
}

// A block takes one row and head; window and landmarks are one list, cut evenly over splits and waves.
template <typename T, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 4) void cache_attn_list_kernel(CacheAttnParams p, int ns) {
    __shared__ float2 ml[kWaves + 1];
    __shared__ float accs[kWaves * D];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int t = blockIdx.x / p.n_heads, h = blockIdx.x - t * p.n_heads, split = blockIdx.y;
    const Row r(p, t);
    List<T, D, 4> list(p, r, h / (p.n_heads / p.c.n_kv));
    const int nwin = max(r.end - r.low + 1, 0), n = r.live ? nwin + p.k_lmk : 0;
    const int per_split = ceil_div(n, ns), i0 = min(split * per_split, n), i1 = min(i0 + per_split, n);
    const int per = (ceil_div(i1 - i0, kWaves) + list.KPW - 1) / list.KPW * list.KPW;
    const int b0 = min(i0 + wv * per, i1), b1 = min(b0 + per, i1);
    const int64_t set = r.live ? ((int64_t)h * p.n_reqs + r.req) * p.k_lmk : 0;
    auto look = [&](int i) {
        const bool lm = i >= nwin && i < b1;
        const int64_t at = lm ? set + i - nwin : -1;
        int j = (int)((unsigned)r.low + (unsigned)i);
        if (lm) j = p.lmk[at];
        return list.place(j, list.page(j, lm ? j < r.low : i < b1), at);
    };
    Slot cur = {kNone, 0.f, 0.f, 0.f};
    if (b0 < b1) cur = look(b0 + lane);
    list.begin((const T*)p.q + (int64_t)t * p.q_st + (int64_t)h * p.q_sh);
    for (int b = b0; b < b1; b += list.NB) {
        const Slot now = cur;
        list.take(now, min(list.NB, b1 - b), [&] {
            if (b + list.NB < b1) cur = look(b + list.NB + lane);
        });
    }
    list.end(ml + wv, accs + wv * D);
    join_parts<T, D, 64 * kWaves>(p, ml, accs, kWaves, 1, 1, t, h, split, ns);
}

// A block takes one row and up to 16 query heads of one key/value head: their window on the matrix cores, then
// each head's landmarks from its list.
template <typename T, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves, (MinWaves<T, D>::value)) void cache_attn_group_kernel(CacheAttnParams p, AttnPlan a) {
    constexpr int QP = Parts<T>::q, PP = Parts<T>::p, KS = D / 32, JN = D / 16, DL = D / 4;
    extern __shared__ float lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, row16 = lane & 15, kg = lane >> 4;
    const int G = p.c.n_kv, group = p.n_heads / G, bt_log = p.c.bt_log, bt = 1 << bt_log;
    const int hx = blockIdx.x % a.tiles, tg = blockIdx.x / a.tiles, g = tg % G, t = tg / G, split = blockIdx.y;
    const int h0 = g * group + hx * 16, nh = min(16, group - hx * 16);
    const bool marks = split < a.nl;
    const int parts = kWaves + (marks ? a.chunks : 0);  // the waves' shares of the window, then chunks of landmarks
    float2* ml = (float2*)lds;
    float* accs = lds + 2 * (kWaves + a.chunks + 1) * a.nh;
    const Row r(p, t);
    const int low = r.low, end = r.end;
    const int32_t* table = r.table;
    const float scale2 = p.scale * kLog2e;
    List<T, D, D / 16> list(p, r, g);

    // the wave's landmarks: chunk c of head hh's slots k0 .. k1; its first 64 are looked up beside the window's pages
    const int kl = marks ? ceil_div(p.k_lmk, a.nl) : 0, k0 = min(split * kl, p.k_lmk), k1 = min(k0 + kl, p.k_lmk);
    const int kc = marks ? ceil_div(k1 - k0, a.chunks) : 0, items = marks ? nh * a.chunks : 0;
    auto slot_at = [&](int i, int hh) { return ((int64_t)(h0 + hh) * p.n_reqs + r.req) * p.k_lmk + i; };
    const int hh1 = wv < items ? wv / a.chunks : 0, c01 = min(k0 + (wv - hh1 * a.chunks) * kc, k1), c11 = min(c01 + kc, k1);
    const bool early = r.live && wv < items && c01 < c11;
    const int64_t at1 = early ? slot_at(min(c01 + lane, c11 - 1), hh1) : 0;
    int j1 = -1;
    if (early && c01 + lane < c11) j1 = p.lmk[at1];
    Slot ahead = {kNone, 0.f, 0.f, 0.f};

    // ---- window: keys base + 32 step ..., from the aligned position at or before the first
    {
        const int base = low & ~(kStep - 1);
        const int steps = r.live && end >= low ? ((end - base) >> 5) + 1 : 0, per = ceil_div(steps, a.ns);
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
        // lane 2 i + half: page (-1: none) of the 16 keys `half` of step i of the batch of 32 steps from b0
        auto look = [&](int b0) {
            const int b = (base + (first + (b0 + (lane >> 1)) * kWaves) * kStep + (lane & 1) * 16) >> bt_log;
            const bool in = b0 + (lane >> 1) < mine && b < p.cols;
            const int page = table[in ? b : 0];
            return in && page >= 0 && page < p.c.n_blocks ? page : -1;
        };
        const int page0 = mine > 0 ? look(0) : -1;
        if (early) ahead = list.place(j1, list.page(j1, j1 < r.low), at1);
        for (int b0 = 0; b0 < mine; b0 += 32) {
            const int page = b0 == 0 ? page0 : look(b0);
            const int64_t tile = (int64_t)max(page, 0) * G + g;
            const float ks = p.c.ks[tile], vs = p.c.vs[tile];
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

    // ---- landmarks
    for (int it = wv; it < items; it += kWaves) {
        const int hh = it / a.chunks, c = it - hh * a.chunks;
        const int c0 = min(k0 + c * kc, k1), c1 = r.live ? min(c0 + kc, k1) : c0;
        auto look = [&](int i) {
            const int64_t at = slot_at(min(i, c1 - 1), hh);
            const int j = i < c1 ? p.lmk[at] : -1;
            return list.place(j, list.page(j, j < low), at);
        };
        list.begin((const T*)p.q + (int64_t)t * p.q_st + (int64_t)(h0 + hh) * p.q_sh);
        Slot cur = ahead;
        if (it != wv && c0 < c1) cur = look(c0 + lane);
        for (int b = c0; b < c1; b += list.NB) {
            const Slot now = cur;
            list.take(now, min(list.NB, c1 - b), [&] {
                if (b + list.NB < c1) cur = look(b + list.NB + lane);
            });
        }
        const int slot = (kWaves + c) * a.nh + hh;
        list.end(ml + slot, accs + slot * D);
    }
    join_parts<T, D, 64 * kWaves>(p, ml, accs, parts, a.nh, nh, t, h0, split, a.ns);
}

// The splits of a row and head joined: a block each, its waves over the splits, a lane D / 64 elements.
constexpr int kJoinWaves = 8;

template <typename T, int D>
__global__ __launch_bounds__(64 * kJoinWaves) void cache_attn_join_kernel(CacheAttnParams p, int ns) {
    constexpr int E = D / 64;
    typedef float vec __attribute__((ext_vector_type(E)));
    __shared__ vec outs[kJoinWaves][64];
    __shared__ float sums[kJoinWaves];
    const int64_t th = blockIdx.x;
    const int t = (int)(th / p.n_heads), h = (int)(th - (int64_t)t * p.n_heads), lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const float2* ml = (const float2*)p.ws + th * ns;
    const float* acc = (const float*)p.ws + 2 * (int64_t)p.n_rows * p.n_heads * ns + th * ns * D + lane * E;
    float M = -INFINITY, L = 0.f;
    for (int k = lane; k < ns; k += 64) M = fmaxf(M, ml[k].x);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, wave_xor(M, o));
    const float mb = M == -INFINITY ? 0.f : M;
    vec o = {};
#pragma unroll 4
    for (int k = wv; k < ns; k += kJoinWaves) {
        const float2 v = ml[k];
        const vec x = *(const vec*)(acc + (int64_t)k * D);
        const float f = v.x == -INFINITY ? 1.f : exp2_(v.x - mb);
        L += v.y == 0.f ? 0.f : v.y * f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += v.y == 0.f ? 0.f : x[e] * f;  // (a split with sum 0 wrote no values)
    }
    outs[wv][lane] = o;
    if (lane == 0) sums[wv] = L;
    __syncthreads();
    if (wv == 0) {
        for (int k = 1; k < kJoinWaves; ++k) {
            o += outs[k][lane];
            L += sums[k];
        }
        T* y = (T*)p.out + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = from_float<T>(L == 0.f ? 0.f : o[e] / L);
        if (lane == 0) p.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
}

// Which kernel, with how many waves and splits.  us on the device, 16/2 heads of 128, 128 landmarks:
//  * A block a head reads a window once for each query head, a block a group once: the former is latency bound and
//    smaller, so it wins up to about 2^18 pairs of a query head and a window key (w_max 512: one request 9 / 19, 8:
//    9 / 21, 32: 17 / 21, 256: 67 / 36; w_max 1024: 8 requests 16 / 23, 24: 27 / 24; w_max 4096, 8 requests: 32 / 23),
//    and where no two query heads share a window.  With each row's whole window of 512: 16 requests 14 / 21, 32: 22 / 22,
//    33: 23 / 22, 48: 27 / 23, 64: 31 / 23, 128: 55 / 28, 256: 102 / 44; float16 and float32 within 2 us of these.
//  * Lists: eight waves for 64 KB of keys or more while there are at most two blocks a CU (one request 9 / 10; 60 requests
//    of 16/16 heads 27 / 23 with four), and four waves with splits of at least 256 keys past 128 KB (one request,
//    w_max 1024: 11 / 14, 4096: 11 / 16).
//  * Groups: eight waves where there is a block a CU at most (64 requests of 8/2 heads 16 / 18, 120 of 16/2 with 512
//    landmarks 45 / 64; 256 of 16/2 43 / 36 with four); windows are split, into 512 keys or more, to one block a CU
//    (four windows of 131072: 32 splits 55, 64 60, 16 71).
AttnPlan attn_plan(const CacheAttnParams& p) {
    AttnPlan a;
    const int group = p.n_heads / p.c.n_kv, D = p.c.head_dim;
    const int64_t cap = (int64_t)p.cols << p.c.bt_log;
    const int64_t w = p.w_max > 0 && p.w_max < cap ? p.w_max : cap;
    const int64_t rows = std::max(p.n_rows, 1);  // (the workspace of a call without rows is asked for too)
    int64_t ns = 1;
    a.list = group == 1 || rows * p.n_heads * w <= 1 << 18;
    if (a.list) {
        const int64_t blocks = rows * p.n_heads, bytes = (w + p.k_lmk) * D;
        a.tiles = group;
        a.nh = 1;
        a.waves = bytes >= 1 << 16 && bytes <= 1 << 17 && blocks <= 512 ? 8 : 4;
        if (bytes > 1 << 17) ns = std::min(1024 / blocks, w / 256);
    } else {
        a.tiles = ceil_div(group, 16);
        a.nh = std::min(group, 16);
        const int64_t blocks = rows * p.c.n_kv * a.tiles;
        a.waves = blocks <= 256 ? 8 : 4;
        ns = std::min(256 / blocks, w / 512);
    }
    a.ns = (int)std::max(ns, (int64_t)1);
    a.nl = std::min(ceil_div(p.k_lmk, 64), a.ns);
    a.chunks = p.k_lmk == 0 ? 0 : std::max(a.waves / a.nh, 1);
    return a;
}

template <typename T, int D>
hipError_t run_rows(const CacheAttnParams& p, const AttnPlan& a, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)p.n_rows * p.c.n_kv * a.tiles), (unsigned)a.ns);
    if (a.list) {
        auto kernel = a.waves == 8 ? cache_attn_list_kernel<T, D, 8> : cache_attn_list_kernel<T, D, 4>;
        DSALT_LAUNCH("cache_attn_list", kernel, grid, dim3(64 * a.waves), 0, stream, p, a.ns);
    } else {
        const unsigned lds = (unsigned)(((a.waves + a.chunks) * (D + 2) + 2) * a.nh * sizeof(float));
        auto kernel = a.waves == 8 ? cache_attn_group_kernel<T, D, 8> : cache_attn_group_kernel<T, D, 4>;
        if (lds > 65536)
            if (hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)) return e;
        DSALT_LAUNCH("cache_attn_group", kernel, grid, dim3(64 * a.waves), lds, stream, p, a);
    }
    if (a.ns > 1) {
        const dim3 join((unsigned)((int64_t)p.n_rows * p.n_heads));
        DSALT_LAUNCH("cache_attn_join", (cache_attn_join_kernel<T, D>), join, dim3(64 * kJoinWaves), 0, stream, p, a.ns);
    }
    return hipGetLastError();
}

template <typename T, int D>
hipError_t run(const CacheAttnParams& p, hipStream_t stream) {
    const AttnPlan a = attn_plan(p);
    const int most = (int)(kLaunchThreads / 256 / (p.c.n_kv * a.tiles));  // rows of a launch (more than one launch: blocks of four waves, no splits)
    CacheAttnParams s = p;
    for (int t = 0; t < p.n_rows; t += s.n_rows) {
        s.n_rows = std::min(most, p.n_rows - t);
        s.q = (const T*)p.q + (int64_t)t * p.q_st;
        s.out = (T*)p.out + (int64_t)t * p.o_st;
        s.lse = p.lse + (int64_t)t * p.n_heads;
        s.req = p.req + t;
        s.pos = p.pos + t;
        s.w = p.w + t;
        if (hipError_t e = run_rows<T, D>(s, a, stream)) return e;
    }
    return hipSuccess;
}

}  // namespace

size_t cache_attn_ws_bytes(const CacheAttnParams& p) {
    const AttnPlan a = attn_plan(p);
    return a.ns > 1 ? (size_t)p.n_rows * p.n_heads * a.ns * (p.c.head_dim + 2) * sizeof(float) : 0;
}

hipError_t cache_attn_launch(const CacheAttnParams& p, hipStream_t stream) {
    if (p.n_rows == 0) return hipSuccess;
    const bool wide = p.c.head_dim == 128;
    switch (p.dtype) {
        case 0: return wide ? run<float, 128>(p, stream) : run<float, 64>(p, stream);
        case 1: return wide ? run<bf16, 128>(p, stream) : run<bf16, 64>(p, stream);
        default: return wide ? run<f16, 128>(p, stream) : run<f16, 64>(p, stream);
    }
}

}  // namespace dsalt
