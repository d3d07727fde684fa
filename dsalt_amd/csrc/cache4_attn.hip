// Attention of query tokens over the paged 4-bit cache: row t is the token at position pos[t] of request req[t] and
// attends A(i) = [i - w + 1, i] U {landmarks p of its head's set : 0 <= p < i - w + 1}.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j + b_j - m): one pass with a running maximum m and sum.  A
// step takes 32 keys: their codes become bfloat16 operands with the scales taken in (exact), and both products run on the
// matrix cores, with up to 16 columns of queries.  Columns of a window are the query heads that share a key/value head, of
// one row or of rows of one request side by side (drafted tokens); columns of a head's landmarks, which are its own, are those rows.
// Scores, weights and sums are kept in 32 bits.
#include <algorithm>

#include "cache4.h"
#include "common.h"
#include "decode_attn.h"
#include "fp4.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kStep = 32;  // keys of a step
constexpr uint32_t kNone = 0xffffffffu;

struct AttnPlan {
    int nh, tiles;      // heads of a block, blocks of a key/value head's query heads
    int nr, run_tiles;  // rows of a block, blocks of a request's rows
    int ns, nl;         // splits of a row's window, and of its landmark slots
    int waves, chunks;  // of a block; parts of a head's landmark slots within a block
    int cols() const { return nr * nh; }
};

template <typename T, int D>
struct Step {  // one wave's running maximum, sum and weighted values of 16 columns
    static constexpr int QP = Parts<T>::q, PP = Parts<T>::p, KS = D / 32, JN = D / 16, DL = D / 4, KW = DL / 8;
    typedef uint32_t kword __attribute__((ext_vector_type(KW)));
    struct Keys {  // lane (row16, kg): elements kg DL ... of keys 16 half + row16
        kword code[2];
        uint32_t scale[2];
    };
    struct Values {  // elements JN row16 ... of keys 16 (e / 4) + 4 kg + e % 4
        uint32_t code[8], scale[8];
    };
    bf16x8 qf[KS][QP];
    floatx4 acc[JN];
    float m, l;

    // the lane's query: column row16, elements kg DL + 8 s + e of step s
    __device__ __forceinline__ void begin(const T* q, int kg) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8];
            load8(q + kg * DL + 8 * s, x);
            split8<QP>(x, qf[s]);
        }
#pragma unroll
        for (int j = 0; j < JN; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.f;
    }
    __device__ __forceinline__ static void load_key(const Cache4Pages& c, uint64_t token, int kg, kword& code, uint32_t& scale) {
        code = *(const kword*)(c.kv + token * D + kg * (DL / 2));
        scale = c.scale[token * (D / 16) + kg * DL / 32];
    }
    __device__ __forceinline__ static void load_value(const Cache4Pages& c, uint64_t token, int row16, uint32_t& code, uint32_t& scale) {
        const uint8_t* x = c.kv + token * D + D / 2 + row16 * (JN / 2);
        code = JN == 8 ? *(const uint32_t*)x : *(const uint16_t*)x;
        scale = c.scale[token * (D / 16) + D / 32 + row16 * JN / 32];
    }
    // scores of keys 16 half + 4 kg + r for column row16
    __device__ __forceinline__ void scores(const Keys& k, float* x) const {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            floatx4 sc = {0.f, 0.f, 0.f, 0.f};
            const float scale = e8m0(k.scale[half]);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const bf16x8 kf = e2m1_op(k.code[half][s], scale);
#pragma unroll
                for (int i = 0; i < QP; ++i) sc = mma(kf, qf[s][i], sc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * half + r] = sc[r];
        }
    }
    // weighted values of the step's keys added to `to`
    __device__ __forceinline__ static void product(const Values& v, const bf16x8* pf, floatx4* to) {
        float scale[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) scale[e] = e8m0(v.scale[e]);
#pragma unroll
        for (int j = 0; j < JN; j += 2) {
            uint32_t c[8];  // elements j and j + 1 of a key
#pragma unroll
            for (int e = 0; e < 8; ++e)
                c[e] = j == 0 ? e2m1_bf16<0>(v.code[e], scale[e])
                     : j == 2 ? e2m1_bf16<1>(v.code[e], scale[e])
                     : j == 4 ? e2m1_bf16<2>(v.code[e], scale[e])
                              : e2m1_bf16<3>(v.code[e], scale[e]);
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{half_pair(c[0], c[1], hi), half_pair(c[2], c[3], hi),
                                                                   half_pair(c[4], c[5], hi), half_pair(c[6], c[7], hi)});
#pragma unroll
                for (int i = 0; i < PP; ++i) to[j + hi] = mma(vf, pf[i], to[j + hi]);
            }
        }
    }
    // The step's scores in base 2 (-inf: masked) and values.  `mixed`: rows of the block's columns see different keys, so
    // that values which are not finite are multiplied row by row: sees(e, r) tells whether row r sees the lane's key e.
    template <typename F>
    __device__ __forceinline__ void take(float* x, const Values& v, bool mixed, int rows, int my_row, F sees) {
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
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = exp2_(x[e] - mb);
            l += x[e];
        }
        bf16x8 pf[PP];
        split8<PP>(x, pf);
        if (mixed) {
            bool nan = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) nan |= v.scale[e] == 255u;
            if (__any(nan)) {
#pragma unroll 1
                for (int r = 0; r < rows; ++r) {
                    Values u = v;
                    floatx4 one[JN];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (!sees(e, r)) u.code[e] = 0u, u.scale[e] = 127u;
#pragma unroll
                    for (int j = 0; j < JN; ++j) one[j] = floatx4{0.f, 0.f, 0.f, 0.f};
                    product(u, pf, one);
#pragma unroll
                    for (int j = 0; j < JN; ++j)
                        if (my_row == r) acc[j] += one[j];
                }
                return;
            }
        }
        product(v, pf, acc);
    }
    // the wave's part of column row16: (maximum, sum) and, where it took any keys, the weighted values [D]
    __device__ __forceinline__ void end(float2* ml, float* out, int kg, bool column, bool any) {
        const float sum = sum_g4(l);
        if (!column) return;
        if (kg == 0) *ml = make_float2(m, sum);
        if (any) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < JN; ++j) out[kg * DL + r * JN + j] = acc[j][r];
        }
    }
};

// The parts of a block's columns joined (ml and accs [part][stride columns]; column c is head c % nh of row c / nh):
// written out, or to the workspace where the row is split.  A part with sum 0 attended nothing and left no values.
template <typename T, int D, int THREADS>
__device__ void join_columns(const Cache4AttnParams& p, float2* ml, const float* accs, int parts, int stride, int n, int nh, int t0, int h0,
                             int split, int ns) {
    float2* total = ml + parts * stride;  // maximum and sum of each column
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += THREADS) {
        float M = -INFINITY, L = 0.f;
        for (int k = 0; k < parts; ++k) M = fmaxf(M, ml[k * stride + c].x);
        const float mb = M == -INFINITY ? 0.f : M;
        for (int k = 0; k < parts; ++k) {
            const float2 v = ml[k * stride + c];
            const float f = v.x == -INFINITY ? 1.f : exp2_(v.x - mb);
            if (v.y != 0.f) L += v.y * f;
            ml[k * stride + c].x = f;
        }
        total[c] = make_float2(M, L);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * D; i += THREADS) {
        const int c = i / D, d = i - c * D, row = c / nh, h = h0 + c - row * nh;
        float o = 0.f;
        for (int k = 0; k < parts; ++k) {
            const float2 v = ml[k * stride + c];
            if (v.y != 0.f) o += accs[(k * stride + c) * D + d] * v.x;
        }
        const float M = total[c].x, L = total[c].y;
        const int64_t th = (int64_t)(t0 + row) * p.n_heads + h;
        if (ns > 1) {
            const int64_t at = th * ns + split;
            if (d == 0) ((float2*)p.ws)[at] = make_float2(M, L);
            if (L != 0.f) ((float*)p.ws)[2 * (int64_t)p.n_rows * p.n_heads * ns + at * D + d] = o;
        } else {
            ((T*)p.out)[(int64_t)(t0 + row) * p.o_st + (int64_t)h * p.o_sh + d] = from_float<T>(L == 0.f ? 0.f : o / L);
            if (d == 0) p.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        }
    }
}

struct Slot {  // a landmark: page, head and token in one number (kNone: not attended), its position and bias in base 2
    uint32_t key;
    int pos;
    float bias;
};

constexpr int kSlots = 64;  // landmarks looked up at a time, a lane each

// A block takes rows of one request, side by side, and query heads of one key/value head, 16 columns at most: their
// window, then each head's landmarks.
template <typename T, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void cache4_attn_kernel(Cache4AttnParams p, AttnPlan a) {
    typedef Step<T, D> S;
    extern __shared__ float lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, row16 = lane & 15, kg = lane >> 4;
    const int G = p.c.n_kv, group = p.n_heads / G, bt_log = p.c.bt_log, bt = 1 << bt_log;
    const int hx = blockIdx.x % a.tiles, tg = blockIdx.x / a.tiles, g = tg % G, rt = tg / G, split = blockIdx.y;
    const int h0 = g * group + hx * a.nh, nh = min(a.nh, group - hx * a.nh);
    const bool marks = split < a.nl;
    const int parts = kWaves + (marks ? a.chunks : 0), stride = a.nr * a.nh;
    float2* ml = (float2*)lds;
    float* accs = lds + 2 * (kWaves + a.chunks + 1) * stride;
    Slot* slots = (Slot*)(accs + (kWaves + a.chunks) * stride * D) + wv * kSlots;
    const float scale2 = p.scale * kLog2e;
    const int run = rt / a.run_tiles;
    const int64_t t_first = (int64_t)run * p.per + (int64_t)(rt - run * a.run_tiles) * a.nr;
    const int64_t t_end = min(min(t_first + a.nr, ((int64_t)run + 1) * p.per), (int64_t)p.n_rows);
    S s;

    for (int64_t tt = t_first; tt < t_end;) {  // (once, unless the rows side by side belong to several requests)
        const int t0 = (int)tt, req = p.req[t0];
        int n = 1;
        while (tt + n < t_end && p.req[t0 + n] == req) ++n;
        tt += n;
        const bool known = req >= 0 && req < p.n_reqs;
        const int32_t* table = p.table + (known ? (int64_t)req * p.table_st : 0);
        const int cap = (p.cols << bt_log) - 1;
        // rows: the lane's for columns of the window, and for those of landmarks
        struct Range { int low, end; };  // first and last key of the window; a row without keys sees nothing
        auto range = [&](int row) {
            const int pos = p.pos[t0 + row];
            const bool live = known && pos >= 0;
            return Range{live ? max(pos - max(p.w[t0 + row], 1) + 1, 0) : 0x7fffffff, live ? min(pos, cap) : -1};
        };
        const int col = row16 < n * nh ? row16 : 0, wrow = col / nh, lrow = row16 < n ? row16 : 0;
        const Range win = range(wrow), mark = range(lrow);
        const int mark_low = mark.low == 0x7fffffff ? 0 : mark.low;
        const int low_min = __builtin_amdgcn_readfirstlane(row_min16(win.low)), low_max = __builtin_amdgcn_readfirstlane(row_max16(win.low));
        const int end_min = __builtin_amdgcn_readfirstlane(row_min16(win.end)), end_max = __builtin_amdgcn_readfirstlane(row_max16(win.end));

        // ---- window: keys base + 32 step ..., from the aligned position at or before the first
        {
            const int base = low_min & ~(kStep - 1);
            const int steps = end_max >= low_min ? ((end_max - base) >> 5) + 1 : 0, per = ceil_div(steps, a.ns);
            const int s0 = split * per, s1 = min(steps, s0 + per);
            s.begin((const T*)p.q + (int64_t)(t0 + wrow) * p.q_st + (int64_t)(h0 + col - wrow * nh) * p.q_sh, kg);
            const int first = s0 + wv, mine = first < s1 ? (s1 - 1 - first) / kWaves + 1 : 0;
            // lane 2 i + half: page (-1: none) of the 16 keys `half` of step i of the batch of 32 steps from b0
            auto look = [&](int b0) {
                const int b = (base + (first + (b0 + (lane >> 1)) * kWaves) * kStep + (lane & 1) * 16) >> bt_log;
                const bool in = b0 + (lane >> 1) < mine && b < p.cols;
                const int page = table[in ? b : 0];
                return in && page >= 0 && page < p.c.n_blocks ? page : -1;
            };
            for (int b0 = 0; b0 < mine; b0 += 32) {
                const int page = look(b0), m = min(32, mine - b0);
                auto token_at = [&](int i, int half) -> uint64_t {  // of the first of 16 keys (page 0 where there is none)
                    const int pg = max(__builtin_amdgcn_readlane(page, 2 * i + half), 0);
                    const int at = base + (first + (b0 + i) * kWaves) * kStep + half * 16;
                    return (((uint64_t)pg * G + g) << bt_log) + (at & (bt - 1));
                };
                typename S::Keys k;
                typename S::Values v;
                auto load_k = [&](int i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) S::load_key(p.c, token_at(i, half) + row16, kg, k.code[half], k.scale[half]);
                };
                auto load_v = [&](int i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint64_t token = token_at(i, half) + 4 * kg;
#pragma unroll
                        for (int e = 0; e < 4; ++e) S::load_value(p.c, token + e, row16, v.code[4 * half + e], v.scale[4 * half + e]);
                    }
                };
                load_k(0);
                load_v(0);
                for (int i = 0; i < m; ++i) {
                    const int at = base + (first + (b0 + i) * kWaves) * kStep;
                    const int pg0 = __builtin_amdgcn_readlane(page, 2 * i), pg1 = __builtin_amdgcn_readlane(page, 2 * i + 1);
                    float x[8];
                    s.scores(k, x);
                    if (i + 1 < m) load_k(i + 1);
                    const bool whole = at >= low_max && at + kStep - 1 <= end_min && pg0 >= 0 && pg1 >= 0;
                    auto key = [&](int e) { return at + (e & 4) * 4 + 4 * kg + (e & 3); };
                    auto held = [&](int e) { return (e < 4 ? pg0 : pg1) >= 0; };
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] *= scale2;
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int j = key(e);
                            if (j < win.low || j > win.end || !held(e)) x[e] = -INFINITY;
                            if (j < low_min || j > end_max || !held(e)) v.code[e] = 0u, v.scale[e] = 127u;  // no column's
                        }
                    }
                    s.take(x, v, !whole && n > 1, n, wrow, [&](int e, int r) {
                        const int j = key(e);
                        // (lanes differ in what they have compared so far, so that none of them may be asked by a shuffle)
                        return j >= __builtin_amdgcn_readlane(win.low, r * nh) && j <= __builtin_amdgcn_readlane(win.end, r * nh) && held(e);
                    });
                    if (i + 1 < m) load_v(i + 1);
                }
            }
            s.end(ml + wv * stride + row16, accs + (wv * stride + row16) * D, kg, row16 < n * nh, mine > 0);
        }

        // ---- landmarks: item (head hh, chunk c) of slots c0 .. c1
        const int kl = marks ? ceil_div(p.k_lmk, a.nl) : 0, k0 = min(split * kl, p.k_lmk), k1 = min(k0 + kl, p.k_lmk);
        const int kc = marks ? ceil_div(k1 - k0, a.chunks) : 0, items = marks ? nh * a.chunks : 0;
        for (int it = wv; it < items; it += kWaves) {
            const int hh = it / a.chunks, c = it - hh * a.chunks;
            const int c0 = min(k0 + c * kc, k1), c1 = known ? min(c0 + kc, k1) : c0;
            s.begin((const T*)p.q + (int64_t)(t0 + lrow) * p.q_st + (int64_t)(h0 + hh) * p.q_sh, kg);
            for (int b = c0; b < c1; b += kSlots) {
                {  // the lane's slot
                    Slot sl = {kNone, 0, 0.f};
                    if (b + lane < c1) {
                        const int64_t at = ((int64_t)(h0 + hh) * p.n_reqs + req) * p.k_lmk + b + lane;
                        sl.pos = p.lmk[at];
                        const int pb = sl.pos >> bt_log;
                        if (sl.pos >= 0 && pb < p.cols) {
                            const int page = table[pb];
                            if (p.lbias) sl.bias = p.lbias[at];
                            if (page >= 0 && page < p.c.n_blocks && sl.bias != -INFINITY) {
                                sl.key = (((uint32_t)page * (uint32_t)G + (uint32_t)g) << bt_log) + (uint32_t)(sl.pos & (bt - 1));
                                // (the type's lowest values stay finite, as masks of them are apart from minus infinity)
                                if (sl.bias > -INFINITY) sl.bias = fmaxf(sl.bias * kLog2e, -3e38f);
                            }
                        }
                    }
                    __builtin_amdgcn_wave_barrier();
                    slots[lane] = sl;
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
                const int steps = ceil_div(min(kSlots, c1 - b), kStep);
                for (int i = 0; i < steps; ++i) {
                    typename S::Keys k;
                    typename S::Values v;
                    Slot sl[8];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t key = slots[i * kStep + half * 16 + row16].key;
                        k.code[half] = typename S::kword{};
                        k.scale[half] = 127u;
                        if (key != kNone) S::load_key(p.c, key, kg, k.code[half], k.scale[half]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        sl[e] = slots[i * kStep + (e & 4) * 4 + 4 * kg + (e & 3)];
                        v.code[e] = 0u;
                        v.scale[e] = 127u;
                        if (sl[e].key != kNone) S::load_value(p.c, sl[e].key, row16, v.code[e], v.scale[e]);
                    }
                    float x[8];
                    s.scores(k, x);
                    auto seen = [&](int e, int low) { return sl[e].key != kNone && sl[e].pos < low; };
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = seen(e, mark_low) ? x[e] * scale2 + sl[e].bias : -INFINITY;
                        if (n == 1 && !seen(e, mark_low)) v.code[e] = 0u, v.scale[e] = 127u;
                    }
                    s.take(x, v, n > 1, n, lrow, [&](int e, int r) { return seen(e, __builtin_amdgcn_readlane(mark_low, r)); });
                }
            }
            const int at = (kWaves + c) * stride + row16 * nh + hh;
            s.end(ml + at, accs + (int64_t)at * D, kg, row16 < n, c0 < c1);
        }
        join_columns<T, D, 64 * kWaves>(p, ml, accs, parts, stride, n * nh, nh, t0, h0, split, a.ns);
        __syncthreads();
    }
}

AttnPlan attn_plan(const Cache4AttnParams& p) {
    AttnPlan a;
    const int group = p.n_heads / p.c.n_kv;
    const int64_t cap = (int64_t)p.cols << p.c.bt_log;
    const int64_t w = p.w_max > 0 && p.w_max < cap ? p.w_max : cap;
    const int64_t rows = std::max(p.n_rows, 1);  // (the workspace of a call without rows is asked for too)
    a.nh = std::min(group, 16);
    a.nr = std::min(p.per, 16 / a.nh);
    a.run_tiles = ceil_div(p.per, a.nr);
    const int64_t groups = (rows + p.per - 1) / p.per * a.run_tiles * p.c.n_kv;
    while (a.nh > 1 && groups * ceil_div(group, a.nh) < 256) a.nh = ceil_div(a.nh, 2);
    a.tiles = ceil_div(group, a.nh);
    const int64_t blocks = groups * a.tiles;
    a.waves = blocks <= 256 ? 8 : 4;
    a.ns = (int)std::max(std::min(512 / blocks, w / 1024), (int64_t)1);
    a.nl = std::min(ceil_div(p.k_lmk, 64), a.ns);
    a.chunks = p.k_lmk == 0 ? 0 : std::max(a.waves / a.nh, 1);
    return a;
}

template <typename T, int D>
hipError_t run_rows(const Cache4AttnParams& p, const AttnPlan& a, hipStream_t stream) {
    const int64_t runs = ((int64_t)p.n_rows + p.per - 1) / p.per;
    const dim3 grid((unsigned)(runs * a.run_tiles * p.c.n_kv * a.tiles), (unsigned)a.ns);
    const unsigned lds = (unsigned)((((a.waves + a.chunks) * (D + 2) + 2) * a.cols()) * sizeof(float) + a.waves * kSlots * sizeof(Slot));
    auto kernel = a.waves == 8 ? cache4_attn_kernel<T, D, 8> : cache4_attn_kernel<T, D, 4>;
    if (lds > 65536)
        if (hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)) return e;
    DSALT_LAUNCH("cache4_attn", kernel, grid, dim3(64 * a.waves), lds, stream, p, a);
    if (a.ns > 1) {
        const dim3 join((unsigned)((int64_t)p.n_rows * p.n_heads));
        DSALT_LAUNCH("cache4_attn_join", (cache_attn_join_kernel<T, D, Cache4AttnParams>), join, dim3(64 * kJoinWaves), 0, stream, p, a.ns);
    }
    return hipGetLastError();
}

template <typename T, int D>
hipError_t run(const Cache4AttnParams& p, hipStream_t stream) {
    const AttnPlan a = attn_plan(p);
    // runs of rows of a launch (more than one launch: blocks of four waves, no splits)
    const int64_t most = std::max(kLaunchThreads / 256 / ((int64_t)p.c.n_kv * a.tiles * a.run_tiles), (int64_t)1) * p.per;
    Cache4AttnParams s = p;
    for (int64_t t = 0; t < p.n_rows; t += s.n_rows) {
        s.n_rows = (int)std::min(most, p.n_rows - t);
        s.q = (const T*)p.q + t * p.q_st;
        s.out = (T*)p.out + t * p.o_st;
        s.lse = p.lse + t * p.n_heads;
        s.req = p.req + t;
        s.pos = p.pos + t;
        s.w = p.w + t;
        if (hipError_t e = run_rows<T, D>(s, a, stream)) return e;
    }
    return hipSuccess;
}

}  // namespace

size_t cache4_attn_ws_bytes(const Cache4AttnParams& p) {
    const AttnPlan a = attn_plan(p);
    return a.ns > 1 ? (size_t)p.n_rows * p.n_heads * a.ns * (p.c.head_dim + 2) * sizeof(float) : 0;
}

hipError_t cache4_attn_launch(const Cache4AttnParams& p, hipStream_t stream) {
    if (p.n_rows == 0) return hipSuccess;
    const bool wide = p.c.head_dim == 128;
    switch (p.dtype) {
        case 0: return wide ? run<float, 128>(p, stream) : run<float, 64>(p, stream);
        case 1: return wide ? run<bf16, 128>(p, stream) : run<bf16, 64>(p, stream);
        default: return wide ? run<f16, 128>(p, stream) : run<f16, 64>(p, stream);
    }
}

}  // namespace dsalt
