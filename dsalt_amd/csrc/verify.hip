// Drafted tokens taken or refused against the target's probabilities, from given random numbers, and the token after them.
//
// Row t of a request holds the target's logits for the token after tokens[t]; its draft x is tokens[t + 1] (the last row has
// none).  With m a row's largest logit, a token weighs a_j = round(2^42 exp((x_j - m) / temperature)), a whole number, and has
// the probability p_j = a_j / sum a; the draft's logits give b and q alike.  The draft is taken while u q_x < p_x.  At
// the first that is refused the token is drawn from what the draft left of p, round(2^52 max(p_j - q_j, 0)) (from p where that
// is nothing), behind the last from p: the first index whose running sum passes v times the total.  Sums of whole numbers do
// not depend on their order, so that a step's tokens do not depend on how its rows are cut.
//
// Four launches: the largest logit of each part of a row; each part's sum of weights; each request's first refused row (its
// probabilities follow from the sums) and the sums over its chunks of what the token is drawn from; the draw, in the one chunk
// that holds it.  The first reads the rows from memory and is bound by that (91 MB 18 us), the others find them in the caches
// and are bound by the arithmetic of the weights, in float64 (a float32 one is off by 2^-24 of itself, which over a vocabulary
// moves a border of the running sums past v once in some thousand draws), or where those of bfloat16 logits are looked up by
// value, by LDS.  One request of five rows: 4, 6, 7 and 6 us, what a launch and its dependent loads take.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "timing.h"
#include "verify.h"
#include "weights.h"

namespace dsalt {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
typedef unsigned long long u64;

struct VerifyPlan {
    int parts;   // of a row, for its largest logit and its sum
    int chunks;  // of a row: 64 vectors of 16 bytes (the first may begin before the row)
    int spread;  // blocks of a request over the chunks of its drawing row
    bool sum_table, pick_table;  // bfloat16 rows by value
};

// A row of n logits as vectors of 16 bytes, the first of which may begin `shift` elements before it.
template <typename T>
struct Logits {
    static constexpr int VEC = 16 / sizeof(T), CHUNK = 64 * VEC;
    typedef T vec __attribute__((ext_vector_type(VEC), aligned(16)));
    const T* x;
    int n, shift, vecs;
    __device__ __forceinline__ Logits(const void* base, int64_t st, int row, int cols) {
        x = (const T*)base + (int64_t)row * st;
        n = cols;
        shift = (int)(((uintptr_t)x & 15) / sizeof(T));
        vecs = (n + shift + VEC - 1) / VEC;
    }
    __device__ __forceinline__ int first(int i) const { return i * VEC - shift; }
    __device__ __forceinline__ bool inside(int i) const { return first(i) >= 0 && first(i) + VEC <= n; }
    __device__ __forceinline__ u32x4 raw(int i) const { return *(const u32x4*)(x + first(i)); }
    // vector i, elements that lie outside the row as NaN
    __device__ __forceinline__ void load(int i, float* f) const {
        const int at = first(i);
        if (inside(i)) {
            const vec v = *(const vec*)(x + at);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = to_float(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = at + e >= 0 && at + e < n ? to_float(x[at + e]) : NAN;
        }
    }
};

// keys: larger logits, larger keys; NaN as minus infinity, whose key is the least, minus zero as zero
__device__ __forceinline__ uint32_t key_of(float x) {
    uint32_t u = __float_as_uint(x);
    if (x != x) u = 0xff800000u;
    if (u == 0x80000000u) u = 0u;
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key); }

// The weights of a row, from its largest logit and the first index that has it.
struct Weigh {
    double m, rate;
    float low;  // logits from here down weigh nothing
    int first;
    bool greedy, empty;
    bool plain;  // exponents of logits from `low` up are small enough to be formed without bounds
    __device__ __forceinline__ Weigh(u64 top, float temp) {
        const float best = value_of((uint32_t)(top >> 32));
        first = (int)~(uint32_t)top;
        greedy = !(temp > 0.f);
        empty = best == -INFINITY;
        // (beside infinity nothing else weighs)
        m = best == INFINITY ? 1e39 : (double)best;
        rate = best == INFINITY ? 1.0 : 1.4426950408889634 / (double)temp;
        // 2^42 2^-43 rounds to 0; exponents of 96 for `low` itself, which is rounded by half of what lies between, and below m
        low = fminf((float)(m - 96.0 * 0.6931471805599453 * (double)temp), best == 0.f ? -1e-45f : __uint_as_float(__float_as_uint(best) + (best > 0.f ? -1 : 1)));
        plain = !greedy && !empty && best < INFINITY && low > -INFINITY && (m - (double)low) * rate < 1000.0;
    }
    __device__ __forceinline__ u64 of(float v, int i) const {
        if (greedy) return i == first && !empty ? kUnit : 0;
        return whole_weight(fmin(fmax(((double)v - m) * rate, -60.0), 0.0));
    }
    // the same of a plain row (fmaxf takes NaN for `low` too)
    __device__ __forceinline__ u64 fast(float v) const { return whole_weight(((double)fmaxf(v, low) - m) * rate); }
};

// Weights of a plain row's bfloat16 logits by value: few values lie between the largest and `low`, so that each is formed once
// and an element costs a look-up.  An entry a sign and magnitude (the upper bits of the float32) from a0, the second of each
// sign; the last of each sign stands for all beyond, of weight 0.  Magnitudes below a0 (2^-15 of the largest that weighs, and
// always zeros) have each sign's first entry: they are weighed directly.  Entries are whole numbers, or their products
// with a share, in float64.
constexpr int kSide = 2048;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct Table {
    double* w;  // [2 kSide]
    uint32_t a0;
    template <typename F>
    __device__ __forceinline__ Table(double* lds, const Weigh& g, int threads, F of) : w(lds) {
        const float m = (float)g.m;
        const uint32_t up = m > 0.f ? __float_as_uint(m) >> 16 : 0;
        const uint32_t down = g.low < 0.f ? min((__float_as_uint(-g.low) >> 16) + 1, 0x7f7fu) : 0;
        const uint32_t most = max(up, down);
        a0 = most > kSide - 3 ? most - (kSide - 3) : 1;
        for (int i = threadIdx.x; i < 2 * kSide; i += threads) {
            const int in = i & (kSide - 1);
            const float v = __uint_as_float((uint32_t)(i / kSide) << 31 | ((uint32_t)in + a0 - 1) << 16);
            w[i] = in >= 1 && in <= kSide - 2 && v <= m ? of(g.fast(v)) : 0.0;
        }
    }
    // the entries of eight logits, two in a word, and whether one of them is a first one
    struct Entries {
        uint32_t two[4];
        bool first;
    };
    __device__ __forceinline__ Entries entries(u32x4 u) const {
        const u16x2 less = {(uint16_t)(a0 - 1), (uint16_t)(a0 - 1)}, most = {kSide - 1, kSide - 1};
        Entries n;
        u16x2 least = most;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u16x2 in = __builtin_elementwise_min(__builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, u[k] & 0x7fff7fffu), less), most);
            least = __builtin_elementwise_min(least, in);
            n.two[k] = (u[k] >> 4 & 0x08000800u) | __builtin_bit_cast(uint32_t, in);
        }
        n.first = (least[0] == 0) | (least[1] == 0);
        return n;
    }
    __device__ __forceinline__ void values(const Entries& n, double* e) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            e[2 * k] = w[n.two[k] & 0xffffu];
            e[2 * k + 1] = w[n.two[k] >> 16];
        }
    }
    // those of first entries, weighed directly
    template <typename F>
    __device__ __forceinline__ static void direct(const Entries& n, u32x4 u, const Weigh& g, F of, double* e) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if ((n.two[k] & 0x7ff) == 0) e[2 * k] = of(g.fast(__uint_as_float(u[k] << 16)));
            if ((n.two[k] >> 16 & 0x7ff) == 0) e[2 * k + 1] = of(g.fast(__uint_as_float(u[k] & 0xffff0000u)));
        }
    }
};

struct Work {  // the workspace
    u64* top;     // [rows][2][parts] key of the largest logit and the complement of its index
    u64* sum;     // [rows][2][parts]
    u64* chunk;   // [n_reqs][chunks]
    int32_t* at;  // [n_reqs] row drawn from; bit 30: from what its draft left
    __host__ __device__ Work(const VerifyParams& p, const VerifyPlan& a) {
        top = (u64*)p.ws;
        sum = top + (int64_t)p.n_rows * 2 * a.parts;
        chunk = sum + (int64_t)p.n_rows * 2 * a.parts;
        at = (int32_t*)(chunk + (int64_t)p.n_reqs * a.chunks);
    }
};

struct Run {  // rows of a request
    int t0, t1;
    __device__ __forceinline__ Run(const VerifyParams& p, int r) {
        t0 = min(max(p.cu[r], 0), p.n_rows);
        t1 = min(max(p.cu[r + 1], t0), p.n_rows);
    }
};
// the request that holds row t, -1: none
__device__ __forceinline__ int request(const VerifyParams& p, int t) {
    int lo = 0, hi = p.n_reqs;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo < p.n_reqs && p.cu[lo] <= t ? lo : -1;
}
__device__ __forceinline__ float temperature(const VerifyParams& p, int side, int r) {
    return side ? (p.draft_temperature ? p.draft_temperature[r] : p.draft_temperature_all)
                : (p.temperature ? p.temperature[r] : p.temperature_all);
}
__device__ __forceinline__ double uniform(const void* u, int f64, int i) {
    const double x = f64 ? ((const double*)u)[i] : (double)((const float*)u)[i];
    return x >= 0.0 ? x : 0.0;
}

// Sum and maximum over the wave of 64-bit numbers (all lanes get them), by moves between lanes alone: a shuffle through LDS
// takes some hundred cycles a step (pick of one request 21 us with rows' parts added by a thread, 7.7 with shuffles)
template <int CTRL>
__device__ __forceinline__ u64 turned(u64 v) {  // lanes of each sixteen turned
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, false);
    return (u64)hi << 32 | lo;
}
template <typename F>
__device__ __forceinline__ u64 over_wave(u64 v, F both) {
    v = both(v, turned<0x121>(v));
    v = both(v, turned<0x122>(v));
    v = both(v, turned<0x124>(v));
    v = both(v, turned<0x128>(v));
    uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    auto b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = both((u64)(uint32_t)b[0] << 32 | (uint32_t)a[0], (u64)(uint32_t)b[1] << 32 | (uint32_t)a[1]);
    lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    auto c = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    auto d = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return both((u64)(uint32_t)d[0] << 32 | (uint32_t)c[0], (u64)(uint32_t)d[1] << 32 | (uint32_t)c[1]);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
    return over_wave(v, [](u64 x, u64 y) { return x + y; });
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
    return over_wave(v, [](u64 x, u64 y) { return x > y ? x : y; });
}

template <typename F>
__device__ __forceinline__ u64 over_sixteen(u64 v, F both) {
    v = both(v, turned<0x121>(v));
    v = both(v, turned<0x122>(v));
    v = both(v, turned<0x124>(v));
    return both(v, turned<0x128>(v));
}

// block (row, side, part): vectors of the part, and whether the row has a draft (or is a target's)
struct Part {
    int t, side, part, i0, i1, req;
    bool on;
    template <typename T>
    __device__ __forceinline__ Part(const VerifyParams& p, const VerifyPlan& a, const T*) {
        const int sides = p.y ? 2 : 1;
        t = blockIdx.x / sides;
        side = blockIdx.x - t * sides;
        part = blockIdx.y;
        req = request(p, t);
        on = req >= 0 && (side == 0 || t + 1 < Run(p, req).t1);
        const int vecs = (p.n_cols + 2 * Logits<T>::VEC - 2) / Logits<T>::VEC, per = ceil_div(vecs, a.parts);
        i0 = part * per;
        i1 = i0 + per;
    }
    __device__ __forceinline__ int64_t at(const VerifyPlan& a) const { return ((int64_t)t * 2 + side) * a.parts + part; }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_top_kernel(VerifyParams p, VerifyPlan a) {
    __shared__ u64 red[kWaves];
    const Part b(p, a, (const T*)nullptr);
    if (b.side == 0 && b.part == 0 && threadIdx.x == 0) p.out[b.t] = -1;
    if (!b.on) return;
    const Logits<T> x(b.side ? p.y : p.x, b.side ? p.y_st : p.x_st, b.t, p.n_cols);
    float best = -INFINITY;
    int best_at = b.i0;
    const int i1 = min(b.i1, x.vecs);
#pragma unroll 4
    for (int i = b.i0 + (int)threadIdx.x; i < i1; i += kThreads) {
        float f[Logits<T>::VEC];
        x.load(i, f);
        float m = f[0];
#pragma unroll
        for (int e = 1; e < Logits<T>::VEC; ++e) m = fmaxf(m, f[e]);
        best_at = m > best ? i : best_at;
        best = fmaxf(best, m);
    }
    u64 top = (u64)key_of(-INFINITY) << 32;
    if (best > -INFINITY) {
        float f[Logits<T>::VEC];
        x.load(best_at, f);
        int e0 = 0;
#pragma unroll
        for (int e = Logits<T>::VEC - 1; e >= 0; --e) e0 = f[e] == best ? e : e0;
        top = ((u64)key_of(best) << 32) | (uint32_t)~(x.first(best_at) + e0);
    }
    top = wave_max64(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kWaves; ++k) top = red[k] > top ? red[k] : top;
        Work(p, a).top[b.at(a)] = top;
    }
}

constexpr int64_t kMostParts = 64;

// largest logit and sum of a row from its parts, a lane each (all lanes of a wave take part and get them)
__device__ __forceinline__ u64 row_top(const Work& w, const VerifyPlan& a, int t, int side) {
    const int lane = threadIdx.x & 63;
    return wave_max64(lane < a.parts ? w.top[((int64_t)t * 2 + side) * a.parts + lane] : 0);
}
__device__ __forceinline__ u64 row_sum(const Work& w, const VerifyPlan& a, int t, int side) {
    const int lane = threadIdx.x & 63;
    return wave_sum64(lane < a.parts ? w.sum[((int64_t)t * 2 + side) * a.parts + lane] : 0);
}

// The part's sum of weights.  TABLE: bfloat16 rows by value.
constexpr int kTableThreads = 512;

template <typename T, bool TABLE>
__global__ __launch_bounds__(TABLE ? kTableThreads : kThreads) void verify_sum_kernel(VerifyParams p, VerifyPlan a) {
    constexpr int THREADS = TABLE ? kTableThreads : kThreads, VEC = Logits<T>::VEC;
    __shared__ u64 red[THREADS / 64];
    const Part b(p, a, (const T*)nullptr);
    if (!b.on) return;
    const Work w(p, a);
    const Weigh weigh(row_top(w, a, b.t, b.side), temperature(p, b.side, b.req));
    const Logits<T> x(b.side ? p.y : p.x, b.side ? p.y_st : p.x_st, b.t, p.n_cols);
    const int i1 = min(b.i1, x.vecs), i0 = b.i0 + (int)threadIdx.x;
    u64 s = 0;
    if (weigh.greedy || weigh.empty) {
        s = b.part == 0 && threadIdx.x == 0 && !weigh.empty ? kUnit : 0;
    } else if (!weigh.plain) {
        for (int i = i0; i < i1; i += THREADS) {
            float f[VEC];
            x.load(i, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += weigh.of(f[e], 0);
        }
    } else if constexpr (TABLE) {
        __shared__ double table[2 * kSide];
        const Table tab(table, weigh, THREADS, [](u64 v) { return (double)v; });
        __syncthreads();
        // (a thread's sum stays below 2^53: its elements are fewer than 2^11)
        double d = 0.0;
        auto add = [&](u32x4 u) {
            const Table::Entries n = tab.entries(u);
            double e[8];
            tab.values(n, e);
            if (n.first) Table::direct(n, u, weigh, [](u64 v) { return (double)v; }, e);
#pragma unroll
            for (int k = 0; k < 8; ++k) d += e[k];
        };
        auto fetch = [&](int i) { return i < i1 && x.inside(i) ? x.raw(i) : u32x4{} + 0x7fc07fc0u; };  // (NaN weighs nothing)
        u32x4 u0 = fetch(i0), u1 = fetch(i0 + THREADS);
        for (int i = i0; i < i1; i += THREADS) {
            const u32x4 u = u0;
            u0 = u1;
            u1 = fetch(i + 2 * THREADS);
            if (x.inside(i)) {
                add(u);
            } else {  // the row's ends
                float f[VEC];
                x.load(i, f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s += weigh.fast(f[e]);
            }
        }
        s += (u64)d;
    } else {
        for (int i = i0; i < i1; i += THREADS) {
            float f[VEC];
            x.load(i, f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += weigh.fast(f[e]);
        }
    }
    s = wave_sum64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < THREADS / 64; ++k) s += red[k];
        w.sum[b.at(a)] = s;
    }
}

// What a request's token is drawn from: the weights of a row, or what its draft left of them.
template <typename T>
struct Drawn {
    Logits<T> x, y;
    Weigh wx, wy;
    double sx, sy;  // 2^52 over the sums
    int draft;
    bool left, pair;  // of what is left; with the draft's logits
    __device__ __forceinline__ Drawn(const VerifyParams& p, const VerifyPlan& a, const Work& w, int r, int t, bool left_)
        : x(p.x, p.x_st, t, p.n_cols), y(p.y ? p.y : p.x, p.y ? p.y_st : p.x_st, t, p.n_cols), wx(row_top(w, a, t, 0), temperature(p, 0, r)),
          wy(left_ && p.y ? row_top(w, a, t, 1) : 0ull, temperature(p, 1, r)), left(left_), pair(left_ && p.y) {
        auto per = [](u64 total) { return total ? 0x1p52 / (double)total : 0.0; };
        sx = left ? per(row_sum(w, a, t, 0)) : 0.0;
        sy = pair ? per(row_sum(w, a, t, 1)) : 0.0;
        draft = left ? (int)min(max(p.tokens[t + 1], (int64_t)-1), (int64_t)0x7fffffff) : -1;
    }
    __device__ __forceinline__ bool plain() const { return wx.plain && (!pair || (wy.plain && y.shift == x.shift)); }
    // what is left of a weight; q: the draft's share
    __device__ __forceinline__ u64 rest(double a, double q) const { return (u64)rint(fmax(a - q, 0.0)); }
    // the weights of the VEC elements of vector i; 0 outside the row
    __device__ __forceinline__ void weights(int i, u64* g) const {
        constexpr int VEC = Logits<T>::VEC;
        float f[VEC], h[VEC];
        if (plain() && x.inside(i)) {
            x.load(i, f);
            if (pair) y.load(i, h);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                g[e] = wx.fast(f[e]);
                if (left) g[e] = rest((double)g[e] * sx, pair ? (double)wy.fast(h[e]) * sy : x.first(i) + e == draft ? 0x1p52 : 0.0);
            }
            return;
        }
        x.load(i, f);
        if (pair) {  // (the draft's row may begin elsewhere in its vector)
            if (y.shift == x.shift) {
                y.load(i, h);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int j = x.first(i) + e;
                    h[e] = j >= 0 && j < y.n ? to_float(y.x[j]) : NAN;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int j = x.first(i) + e;
            g[e] = wx.of(f[e], j);
            if (left) {
                const double q = pair ? (double)wy.of(h[e], j) * sy : j == draft ? 0x1p52 : 0.0;
                g[e] = rest((double)g[e] * sx, q);
            }
            if (j < 0 || j >= x.n) g[e] = 0;
        }
    }
};

// Block (request, share of the chunks): the first refused row, and the sums of its chunks.  TABLE: bfloat16 rows by value.
constexpr int kPickThreads = 1024;

template <typename T, bool TABLE>
__global__ __launch_bounds__(TABLE ? kPickThreads : kThreads) void verify_pick_kernel(VerifyParams p, VerifyPlan a) {
    constexpr int THREADS = TABLE ? kPickThreads : kThreads, WAVES = THREADS / 64, VEC = Logits<T>::VEC;
    __shared__ double tables[TABLE ? 2 : 1][TABLE ? 2 * kSide : 1];
    int& refused = *(int*)tables;  // (before the tables are there)
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Run run(p, r);
    const Work w(p, a);
    if (tid == 0) refused = run.t1 - 1;
    __syncthreads();
    for (int t = run.t0 + (tid >> 4); t + 1 < run.t1; t += THREADS / 16) {  // sixteen lanes a draft
        const int64_t x = p.tokens[t + 1];
        bool taken = false;
        if (x >= 0 && x < p.n_cols) {
            auto share = [&](int side) {
                const T* row = side ? (const T*)p.y + (int64_t)t * p.y_st : (const T*)p.x + (int64_t)t * p.x_st;
                const float v = to_float(row[x]);
                const int64_t at = ((int64_t)t * 2 + side) * a.parts;
                u64 top = 0, total = 0;
                for (int k = tid & 15; k < a.parts; k += 16) {
                    const u64 y = w.top[at + k];
                    top = y > top ? y : top;
                    total += w.sum[at + k];
                }
                top = over_sixteen(top, [](u64 y, u64 z) { return y > z ? y : z; });
                total = over_sixteen(total, [](u64 y, u64 z) { return y + z; });
                const Weigh g(top, temperature(p, side, r));
                return total ? (double)g.of(v, (int)x) / (double)total : 0.0;
            };
            const double q = p.y ? share(1) : 1.0;
            taken = uniform(p.u, p.u_f64, t) * q < share(0);
        }
        if (!taken && (tid & 15) == 0) atomicMin(&refused, t);
    }
    __syncthreads();
    const int t = __builtin_amdgcn_readfirstlane(refused);
    if (run.t0 >= run.t1) {
        if (tid == 0 && blockIdx.y == 0) w.at[r] = -1;
        return;
    }
    const bool left = t + 1 < run.t1;
    if (tid == 0 && blockIdx.y == 0) w.at[r] = t | (left ? 1 << 30 : 0);
    const Drawn<T> d(p, a, w, r, t, left);
    u64* chunk = w.chunk + (int64_t)r * a.chunks;
    const int c0 = blockIdx.y * WAVES + wv, step = gridDim.y * WAVES;
    if constexpr (TABLE) {
        if (d.plain()) {
            __syncthreads();
            // (what the draft left is a difference of shares, formed from entries that are shares already)
            auto share_a = [&](u64 v) { return left ? (double)v * d.sx : (double)v; };
            auto share_b = [&](u64 v) { return (double)v * d.sy; };
            const Table ta(tables[0], d.wx, THREADS, share_a);
            Table tb = ta;
            if (d.pair) tb = Table(tables[1], d.wy, THREADS, share_b);
            __syncthreads();
            const u32x4 none = u32x4{} + 0x7fc07fc0u;
            auto inside = [&](int c) { return c < a.chunks && d.x.inside(c * 64) && d.x.inside(c * 64 + 63); };
            auto fetch = [&](int c, u32x4& u, u32x4& v) {
                u = v = none;
                if (inside(c)) {
                    u = d.x.raw(c * 64 + lane);
                    if (d.pair) v = d.y.raw(c * 64 + lane);
                }
            };
            u32x4 u0, v0, u1, v1;
            fetch(c0, u0, v0);
            fetch(c0 + step, u1, v1);
            for (int c = c0; c < a.chunks; c += step) {
                const u32x4 u = u0, v = v0;
                u0 = u1, v0 = v1;
                fetch(c + 2 * step, u1, v1);
                double sum = 0.0;
                const bool direct = !inside(c);
                if (!direct) {
                    double e[8], q[8];
                    const Table::Entries n = ta.entries(u);
                    ta.values(n, e);
                    if (n.first) Table::direct(n, u, d.wx, share_a, e);
                    if (left) {
                        if (d.pair) {
                            const Table::Entries o = tb.entries(v);
                            tb.values(o, q);
                            if (o.first) Table::direct(o, v, d.wy, share_b, q);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) q[k] = d.x.first(c * 64 + lane) + k == d.draft ? 0x1p52 : 0.0;
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k) e[k] = rint(fmax(e[k] - q[k], 0.0));
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) sum += e[k];
                }
                u64 s = (u64)sum;
                if (direct) {  // the row's ends
                    u64 g[VEC];
                    d.weights(c * 64 + lane, g);
                    s = 0;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s += g[e];
                }
                s = wave_sum64(s);
                if (lane == 0) chunk[c] = s;
            }
            return;
        }
    }
    for (int c = c0; c < a.chunks; c += step) {
        u64 g[VEC], s = 0;
        d.weights(c * 64 + lane, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += g[e];
        s = wave_sum64(s);
        if (lane == 0) chunk[c] = s;
    }
}

// exclusive prefix of v over the block, and the total
__device__ __forceinline__ u64 block_scan(u64* red, u64 v, u64& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    u64 in = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(in, d);
        if (lane >= d) in += o;
    }
    __syncthreads();
    if (lane == 63) red[wv] = in;
    __syncthreads();
    u64 base = 0;
    total = 0;
    for (int k = 0; k < kWaves; ++k) {
        if (k == wv) base = total;
        total += red[k];
    }
    return base + in - v;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyParams p, VerifyPlan a) {
    constexpr int VEC = Logits<T>::VEC;
    __shared__ u64 red[kWaves], before;
    __shared__ int found;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const Run run(p, r);
    const Work w(p, a);
    if (run.t0 >= run.t1) {
        if (tid == 0) p.accepted[r] = 0;
        return;
    }
    const int at = w.at[r], t = at & ~(1 << 30);
    bool left = at >> 30;
    for (int i = run.t0 + tid; i < t; i += kThreads) p.out[i] = p.tokens[i + 1];
    if (tid == 0) p.accepted[r] = t - run.t0;
    u64* chunk = w.chunk + (int64_t)r * a.chunks;
    Drawn<T> d(p, a, w, r, t, left);
    const int per = ceil_div(a.chunks, kThreads), c0 = min(tid * per, a.chunks), c1 = min(c0 + per, a.chunks);
    u64 cum = 0, total = 0;
    for (int again = 0; again < 2; ++again) {
        u64 s = 0;
        for (int c = c0; c < c1; ++c) s += chunk[c];
        cum = block_scan(red, s, total);
        if (total || !left) break;
        left = false;  // the draft left nothing: the row's own weights
        d = Drawn<T>(p, a, w, r, t, false);
        for (int c = tid >> 6; c < a.chunks; c += kWaves) {
            u64 g[VEC], s1 = 0;
            d.weights(c * 64 + lane, g);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s1 += g[e];
            s1 = wave_sum64(s1);
            if (lane == 0) chunk[c] = s1;
        }
        __syncthreads();
    }
    if (total == 0) return;  // (no logit above minus infinity: -1)
    double goal = uniform(p.v, p.u_f64, r) * (double)total;
    if (!((double)total > goal))  // v >= 1: the last token (the float64 below the total)
        goal = __longlong_as_double(__double_as_longlong((double)total) - 1);
    if (tid == 0) found = -1;
    __syncthreads();
    for (int c = c0; c < c1; ++c) {
        const u64 next = cum + chunk[c];
        if (!((double)cum > goal) && (double)next > goal) {
            found = c;
            before = cum;
        }
        cum = next;
    }
    __syncthreads();
    if (tid < 64 && found >= 0) {
        const int i = found * 64 + lane;
        u64 g[VEC], s = 0;
        d.weights(i, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += g[e];
        u64 in = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u64 y = __shfl_up(in, o);
            if (lane >= o) in += y;
        }
        u64 sum = before + in - s;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (!((double)sum > goal) && (double)(sum + g[e]) > goal) p.out[t] = d.x.first(i) + e;
            sum += g[e];
        }
    }
}

// How rows are cut.  us on the device, 300 rows (182 of 64 requests and 118 of their drafts, 91 MB) of 151936 bfloat16 logits:
//  * By value, 31 for the sums and 22 for what 64 tokens are drawn from, with every weight formed 53 and 35.  A block forms up to
//    4096 entries, so that it takes 12000 logits or more.  1280 blocks for the sums (640 rows: all four launches 128 with 640
//    blocks, 112 with 1920), 256 of 1024 threads for the draw (128: 90, 512: 86, against 78).
//  * With every weight formed: blocks begin with a row's parts and a draft's shares, some hundred instructions, so that there are
//    1024 and 512 of them, not more (37 requests of 9 rows of 50257 float32 logits: 40, with 2048 of each 45).
VerifyPlan verify_plan(const VerifyParams& p) {
    const int vec = p.dtype == 0 ? 4 : 8;
    const int64_t vecs = ((int64_t)p.n_cols + 2 * vec - 2) / vec, rows = (int64_t)std::max(p.n_rows, 1) * (p.y ? 2 : 1);
    const int reqs = std::max(p.n_reqs, 1);
    VerifyPlan a;
    a.chunks = (int)((vecs + 63) / 64);
    const int64_t parts = std::min({1024 / rows, vecs / 512, kMostParts}), spread = std::min((int64_t)(512 / reqs), (int64_t)(a.chunks + kWaves - 1) / kWaves);
    const int64_t by_value = std::clamp(1280 / rows, (int64_t)1, kMostParts), pick_by_value = std::max(256 / reqs, 1);
    // (launches of at most 2^32 - 1 threads)
    a.sum_table = p.dtype == 1 && vecs / by_value >= 1500 && vecs / by_value < (1 << 17) && rows < (1ll << 32) / kTableThreads;
    a.pick_table = p.dtype == 1 && vecs / pick_by_value >= 1500 && reqs < (1ll << 32) / kPickThreads;
    a.parts = (int)std::max(a.sum_table ? by_value : parts, (int64_t)1);
    a.spread = (int)std::max(a.pick_table ? pick_by_value : spread, (int64_t)1);
    return a;
}

template <typename T>
hipError_t run(const VerifyParams& p, hipStream_t stream) {
    constexpr bool by_value = std::is_same_v<T, bf16>;
    const VerifyPlan a = verify_plan(p);
    if (p.n_rows > 0) {
        const dim3 rows((unsigned)p.n_rows * (p.y ? 2u : 1u), (unsigned)a.parts);
        DSALT_LAUNCH("verify_top", verify_top_kernel<T>, rows, dim3(kThreads), 0, stream, p, a);
        if (a.sum_table) DSALT_LAUNCH("verify_sum", (verify_sum_kernel<T, by_value>), rows, dim3(kTableThreads), 0, stream, p, a);
        else DSALT_LAUNCH("verify_sum", (verify_sum_kernel<T, false>), rows, dim3(kThreads), 0, stream, p, a);
    }
    if (p.n_reqs == 0) return hipGetLastError();
    const dim3 picks((unsigned)p.n_reqs, (unsigned)a.spread);
    if (a.pick_table) DSALT_LAUNCH("verify_pick", (verify_pick_kernel<T, by_value>), picks, dim3(kPickThreads), 0, stream, p, a);
    else DSALT_LAUNCH("verify_pick", (verify_pick_kernel<T, false>), picks, dim3(kThreads), 0, stream, p, a);
    DSALT_LAUNCH("verify_draw", verify_draw_kernel<T>, dim3((unsigned)p.n_reqs), dim3(kThreads), 0, stream, p, a);
    return hipGetLastError();
}

}  // namespace

size_t verify_ws_bytes(const VerifyParams& p) {
    const VerifyPlan a = verify_plan(p);
    return (size_t)p.n_rows * 4 * a.parts * sizeof(u64) + (size_t)p.n_reqs * (a.chunks * sizeof(u64) + sizeof(int32_t));
}

hipError_t verify_launch(const VerifyParams& p, hipStream_t stream) {
    switch (p.dtype) {
        case 0: return run<float>(p, stream);
        case 1: return run<bf16>(p, stream);
        default: return run<f16>(p, stream);
    }
}

}  // namespace dsalt
