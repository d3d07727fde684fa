// One token a row of logits, drawn from given random numbers u in [0, 1).
//
// Order the row's tokens by logit, largest first, equal ones by index.  With m the largest logit, a token
// weighs round(2^42 exp((x - m) / temperature)), a whole number: sums of weights do not depend on their
// order, so that a draw is the same whatever the blocks and lanes that form them.  Kept is a prefix of the
// order: the first top_k tokens, of those the ones before which less than top_p of their weight lies, of
// those the ones that weigh at least min_p 2^42.  The token is the first index whose running sum of kept
// weights, in the order of the vocabulary, passes u times the total.
//
// A block takes a row.  With top_k up to 1024 (or a vocabulary up to kList) the few tokens that can be kept
// are listed and sorted.  Otherwise rows of bfloat16 count their values, of which few differ, and rows of other
// types find the end of a prefix in a histogram (of counts for top_k, of weights for top_p) over even parts of the
// weights' exponents: the bins are summed from the top down to the one that holds the end, whose elements are sorted.
//
// A pass over the row reads it from memory once and from the caches after that; what bounds it is the
// arithmetic of one compute unit a row, in float64 where weights are formed (a float32 weight is off by 2^-24
// of itself, which over 150000 tokens moves a border of the running sums past u once in some thousand draws).
// The first pass notes each chunk's largest logit, so that passes over what a filter may keep read few chunks where
// it keeps little (256 rows, top_k 50: 33 us, 43 with every chunk read again).
// us on the device, 256 bfloat16 rows of 151936 (77.8 MB, 15.6 at the copy rate): largest logit 17, top_k 50 33,
// temperature alone 40, top_p 0.9 at temperature 0.5 45, at temperature 2, where most is kept, 67 (73 with an element's
// entry found by itself, 92 with a pass more for the equal elements at the prefix's end).  One row: 9, 27, 28, 33, 52.
// Vector instructions take two thirds of a compute unit's cycles there, look-ups in LDS a third.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "sample.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 4096, kList = 2048;
constexpr double kPerUnit = 94.0;
constexpr unsigned long long kUnit = 1ull << 42;  // sums over 2^20 tokens stay below 2^62

// keys: larger logits, larger keys; 0 where there is no element
template <typename T> struct Key;
template <> struct Key<float> { static constexpr int bits = 32; };
template <> struct Key<bf16> { static constexpr int bits = 16; };  // the upper half of the float32 holds all
template <> struct Key<f16> { static constexpr int bits = 19; };   // sign, 8 exponent and 10 mantissa bits

template <typename T> __device__ __forceinline__ uint32_t key_of(float x) {
    uint32_t u = __float_as_uint(x);
    if (x != x) u = 0xff800000u;      // NaN: as minus infinity
    if (u == 0x80000000u) u = 0u;     // minus zero equals zero
    return (u ^ (u >> 31 ? 0xffffffffu : 0x80000000u)) >> (32 - Key<T>::bits);
}

struct Cut {  // kept: key above, or equal with a lower index
    uint32_t key;
    int idx;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i < idx); }
};

struct Shared {
    unsigned long long bin[kBins + 8];  // histogram bins, or a sum a chunk of the row
    unsigned long long list[kList];     // (2 kThreads) tokens that can be kept: key, then the index's complement
    unsigned long long part[kWaves];
    unsigned long long found[4];
    int count;
    uint16_t top[kBins + 8];            // upper bits of the key of a chunk's largest logit
};

// All of a block's LDS: Shared, then the table of bfloat16 rows.  Dynamic, so that a function that is called rather than
// inlined reaches it by name (through a pointer it would with flat instructions).
extern __shared__ unsigned long long sample_lds[];
__device__ __forceinline__ Shared& shared() { return *(Shared*)sample_lds; }

// exclusive prefix of v over the block, and the total
__device__ __forceinline__ unsigned long long block_scan(Shared& sh, unsigned long long v, unsigned long long& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    unsigned long long in = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long o = __shfl_up(in, d);
        if (lane >= d) in += o;
    }
    __syncthreads();
    if (lane == 63) sh.part[wv] = in;
    __syncthreads();
    unsigned long long base = 0;
    total = 0;
    for (int k = 0; k < kWaves; ++k) {
        if (k == wv) base = total;
        total += sh.part[k];
    }
    return base + in - v;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
// sum over the wave of values whose sum stays below 2^32 (every lane gets it)
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
    v = dpp_add<0x128>(dpp_add<0x124>(dpp_add<0x122>(dpp_add<0x121>(v))));  // rotations within sixteen lanes
    auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = a[0] + a[1];
    auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return b[0] + b[1];
}
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)));
}
// maxima over the wave of four values: lanes 0 to 15 get the first one's, then the third's, the second's and the fourth's
__device__ __forceinline__ float wave_max4(const float* v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[2]), __float_as_uint(v[3]), false, false);
    const float x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])), y = fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
    auto c = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return dpp_max<0x128>(dpp_max<0x124>(dpp_max<0x122>(dpp_max<0x121>(fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]))))));
}
__device__ __forceinline__ uint16_t upper_key(float v) { return (uint16_t)(key_of<bf16>(v)); }
// The same for two values at once, one in each half of the wave after the first step: low + high 2^BITS
template <int BITS>
__device__ __forceinline__ unsigned long long wave_sum2(uint32_t low, uint32_t high) {
    auto a = __builtin_amdgcn_permlane32_swap(low, high, false, false);
    const uint32_t v = dpp_add<0x128>(dpp_add<0x124>(dpp_add<0x122>(dpp_add<0x121>(a[0] + a[1]))));
    auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const int both = (int)(b[0] + b[1]);
    return ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane(both, 32) << BITS) + (uint32_t)__builtin_amdgcn_readlane(both, 0);
}
// and for weights: sums of at most 64 x 8 of 2^42, in two parts of 25 and 20 bits a lane
__device__ __forceinline__ unsigned long long wave_sum_weights(unsigned long long v) {
    return wave_sum2<25>((uint32_t)v & 0x1ffffffu, (uint32_t)(v >> 25));
}

// 2^42 (2^f - 1) = f P(f) for f in [-1/2, 1/2], P the degree 9 polynomial through the ten Chebyshev nodes (relative
// error of 2^f below 2^-50)
__device__ constexpr double kPow2[10] = {0x1.62e42fefa39f7p41, 0x1.ebfbdff82c590p39, 0x1.c6b08d7044119p37, 0x1.3b2ab6fba385fp35,
                                         0x1.5d87fe908f88ap32, 0x1.4309130378460p29, 0x1.ffcb76789860fp25, 0x1.62bfe46117445p22,
                                         0x1.b6571de2f2351p18, 0x1.e5e9f548e5725p14};

// x f + c with c in scalar registers (from vector registers it would be copied before each sum)
__device__ __forceinline__ double fma_s(double x, double f, double c) {
    double y;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(y) : "v"(x), "v"(f), "s"(c));
    return y;
}

template <typename T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T), CHUNK = 64 * VEC;
    typedef T vec __attribute__((ext_vector_type(VEC), aligned(16)));
    typedef const T __attribute__((address_space(1))) global;  // (known to be global memory in called functions too)
    typedef const vec __attribute__((address_space(1))) global_vec;
    global* x;
    int n, shift;  // elements, and those of the first 16-byte vector that lie before the row
    int chunks;
    double m;      // largest logit (beside infinity 1e39, above every other)
    double rate;   // log2(e) / temperature

    // Chunk c: elements c CHUNK - shift ..., VEC a lane from `first`; absent ones are given as NaN.
    __device__ __forceinline__ int first(int c) const { return c * CHUNK + (int)(threadIdx.x & 63) * VEC - shift; }
    __device__ __forceinline__ bool inside(int c) const { return c * CHUNK >= shift && (c + 1) * CHUNK - shift <= n; }
    __device__ __forceinline__ void load(int at, float* v) const {
        if (at >= 0 && at + VEC <= n) {
            const vec u = *(global_vec*)(x + at);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = to_float(u[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = at + e >= 0 && at + e < n ? to_float(x[at + e]) : NAN;
        }
    }
    __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
    // f(chunk, first element of the lane, its VEC values: as floats, or as they are stored where it takes those); r is what
    // was requested of the chunk
    template <typename F>
    __device__ __forceinline__ void give(F f, int c, const vec& r) const {
        if constexpr (std::is_invocable_v<F, int, int, u32x4>) {
            u32x4 u = __builtin_bit_cast(u32x4, r);
            if (!inside(c)) {
                float v[VEC];
                load(first(c), v);
                vec y;
#pragma unroll
                for (int e = 0; e < VEC; ++e) y[e] = (T)v[e];
                u = __builtin_bit_cast(u32x4, y);
            }
            f(c, first(c), u);
        } else {
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = to_float(r[e]);
            if (!inside(c)) load(first(c), v);
            f(c, first(c), v);
        }
    }
    // f (see give) for the wave's chunks, three of them requested ahead
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        auto fetch = [&](int c) {
            vec u = {};
            if (inside(c)) u = *(global_vec*)(x + first(c));
            return u;
        };
        int c = wave();
        vec r0 = fetch(c), r1 = fetch(c + kWaves), r2 = fetch(c + 2 * kWaves);
        for (; c < chunks; c += kWaves) {
            const vec r = r0;
            r0 = r1;
            r1 = r2;
            r2 = fetch(c + 3 * kWaves);
            give(f, c, r);
        }
    }
    // the same for passes of few instructions, which wait for memory: four chunks at a time, the next four requested
    // before they are looked at (and `four` after each four, with the first of them)
    template <typename F>
    __device__ __forceinline__ void skim(F f) const {
        skim(f, [](int) {});
    }
    template <typename F, typename G>
    __device__ __forceinline__ void skim(F f, G four) const {
        constexpr int N = 4;
        auto fetch = [&](int c, vec* r) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                r[k] = vec{};
                if (inside(c + k * kWaves)) r[k] = *(global_vec*)(x + first(c + k * kWaves));
            }
        };
        int c = wave();
        vec r[N], next[N];
        fetch(c, r);
        for (; c < chunks; c += N * kWaves) {
            fetch(c + N * kWaves, next);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int ck = c + k * kWaves;
                if (ck < chunks) give(f, ck, r[k]);
                r[k] = next[k];
            }
            four(c);
        }
    }
    // the same for the chunks whose largest logit may be `low` or more; the others are not read
    template <typename F>
    __device__ __forceinline__ void pick(const uint16_t* top, float low, F f) const {
        constexpr int N = 4;
        const uint32_t least = upper_key(low);
        const int lane = threadIdx.x & 63;
        for (int b = wave(); b < chunks; b += 64 * kWaves) {
            const int mine = b + lane * kWaves;
            unsigned long long left = __ballot(mine < chunks && top[min(mine, chunks - 1)] >= least);
            auto fetch = [&](int* c, vec* r) {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    c[k] = left ? b + __builtin_ctzll(left) * kWaves : -1;
                    left &= left - 1;
                    r[k] = vec{};
                    if (c[k] >= 0 && inside(c[k])) r[k] = *(global_vec*)(x + first(c[k]));
                }
            };
            int c[N], next_c[N];
            vec r[N], next[N];
            fetch(c, r);
            while (c[0] >= 0) {
                fetch(next_c, next);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    if (c[k] >= 0) give(f, c[k], r[k]);
                    c[k] = next_c[k];
                    r[k] = next[k];
                }
            }
        }
    }
    // the one or the other, by the number of such chunks (one row of 151936, top_p 0.9 at temperature 2: 64 us with those
    // picked though most are, 60 with all read)
    template <typename F>
    __device__ __forceinline__ void seek(const uint16_t* top, float low, F f) const {
        const uint32_t least = upper_key(low);
        int n = 0;
        for (int b = wave(); b < chunks; b += 64 * kWaves) {
            const int c = b + (int)(threadIdx.x & 63) * kWaves;
            n += __popcll(__ballot(c < chunks && top[min(c, chunks - 1)] >= least));
        }
        if (2 * kWaves * n < chunks) pick(top, low, f);
        else skim(f);
    }
    __device__ __forceinline__ bool has(int i) const { return (unsigned)i < (unsigned)n; }
    // round(2^42 2^t), t = (v - m) log2(e) / temperature.  (v - m is exact, or rounded to 2^-53 of itself where the two lie
    // far apart; t below -43 rounds to 0, NaN and absent elements among it.  Sums with 1.5 2^52 and 2^52 round to a whole number and leave it in the mantissa.)
    __device__ __forceinline__ unsigned long long weight(float v) const { return weight_of(exponent(v)); }
    __device__ __forceinline__ double exponent(float v) const { return fmin(fmax(((double)v - m) * rate, -60.0), 0.0); }
    __device__ __forceinline__ static unsigned long long weight_of(double t) {
        const double s = t + 6755399441055744.0;
        const double f = t - (s - 6755399441055744.0);
        double y = kPow2[9];
#pragma unroll
        for (int k = 8; k >= 0; --k) y = fma_s(y, f, kPow2[k]);
        y = fma_s(y, f, 0x1p42);
        y = __hiloint2double(__double2hiint(y) + (__double2loint(s) << 20), __double2loint(y)) + 4503599627370496.0;
        return (unsigned long long)__double_as_longlong(y) & 0xfffffffffffffull;
    }
    // The bin of an exponent: kBins even parts of (-43.6, 0], the highest at 0, bin 0 for all beyond (of weight 0).  Rounding
    // keeps the order, so larger logits are never in lower bins.
    __device__ __forceinline__ static int bin_of(double t) { return max(kBins - 1 - (int)(t * -kPerUnit), 0); }
    // bounds of a bin's logits, a rounding or two wider
    __device__ __forceinline__ float below_bin(int b) const { return wider(m - (kBins - b) / kPerUnit / rate, -1.0); }
    __device__ __forceinline__ float above_bin(int b) const {
        return b == kBins - 1 ? INFINITY : wider(m - (kBins - 1 - b) / kPerUnit / rate, 1.0);
    }
    __device__ __forceinline__ float wider(double x, double way) const {
        return (float)(x + way * ((fabs(x) + fabs(m)) * 0x1p-20 + 0x1p-140));
    }
    // the logit of a key
    __device__ __forceinline__ float value(uint32_t key) const {
        constexpr int low = 32 - Key<T>::bits;
        const uint32_t full = key << low;
        return __uint_as_float(full >> 31 ? full ^ 0x80000000u : ~(full | (low ? (1u << low) - 1 : 0u)));
    }
};

// A level of a search: the bins of `width` bits hold amounts; from the top down, the bin b in which
// ends(amount above, its own) holds.  False where none does.
template <typename F>
__device__ __forceinline__ bool find_bin(Shared& sh, int width, unsigned long long above, F ends, unsigned long long& total, uint32_t& bin,
                         unsigned long long& before, unsigned long long& own) {
    const int nb = 1 << width, tid = threadIdx.x;
    unsigned long long h[kBins / kThreads], sum = 0;
#pragma unroll
    for (int e = 0; e < kBins / kThreads; ++e) {
        const int b = nb - 1 - (tid * (kBins / kThreads) + e);
        h[e] = b >= 0 ? sh.bin[b] : 0;
        sum += h[e];
    }
    if (tid == 0) sh.found[0] = ~0ull;
    unsigned long long cum = above + block_scan(sh, sum, total);
#pragma unroll
    for (int e = 0; e < kBins / kThreads; ++e) {
        if (ends(cum, h[e])) {  // one bin at most
            sh.found[0] = (unsigned long long)(nb - 1 - (tid * (kBins / kThreads) + e));
            sh.found[1] = cum;
            sh.found[2] = h[e];
        }
        cum += h[e];
    }
    __syncthreads();
    bin = (uint32_t)sh.found[0];
    before = sh.found[1];
    own = sh.found[2];
    return sh.found[0] != ~0ull;
}

__device__ __forceinline__ void clear_bins(Shared& sh, int n) {
    __syncthreads();
    for (int b = threadIdx.x; b < n; b += kThreads) sh.bin[b] = 0;
    __syncthreads();
}

// the least number, of at most n, of weights w after which a weight of thr is reached
__device__ __forceinline__ unsigned long long reach(unsigned long long above, unsigned long long w, unsigned long long n, double thr) {
    unsigned long long lo = 1, hi = n;
    while (lo < hi) {
        const unsigned long long mid = (lo + hi) >> 1;
        if ((double)(above + mid * w) < thr) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// `cut` moved up to the first `keep` of its `ties` elements of key `prefix`
template <typename T>
__device__ __forceinline__ void keep_equal(Shared& sh, const Row<T>& row, Cut& cut, uint32_t prefix, unsigned long long keep, unsigned long long ties) {
    constexpr int VEC = Row<T>::VEC;
    cut.idx = prefix == cut.key ? cut.idx : 0x7fffffff;
    cut.key = prefix;
    // (which of those at minus infinity, NaN among them, does not matter: they weigh nothing)
    if (keep >= ties || prefix == key_of<T>(-INFINITY)) return;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    // the index of the first one left out
    const float value = row.value(prefix);
    auto tie = [&](float v, int i) { return v == value && i < cut.idx; };
    __syncthreads();
    row.skim([&](int c, int at, const float* v) {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) n += tie(v[e], at + e);
        n = wave_sum(n);
        if (lane == 0) sh.bin[c] = n;
    });
    __syncthreads();
    const int per = ceil_div(row.chunks, kThreads), c0 = min(tid * per, row.chunks), c1 = min(c0 + per, row.chunks);
    unsigned long long sum = 0, total;
    for (int c = c0; c < c1; ++c) sum += sh.bin[c];
    unsigned long long cum = block_scan(sh, sum, total);
    for (int c = c0; c < c1; ++c) {
        if (cum <= keep && keep < cum + sh.bin[c]) {
            sh.found[0] = c;
            sh.found[1] = cum;
        }
        cum += sh.bin[c];
    }
    __syncthreads();
    if (wv == 0) {
        const int at = row.first((int)sh.found[0]);
        float v[VEC];
        row.load(at, v);
        int n = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) n += tie(v[e], at + e);
        int in = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        int before = (int)sh.found[1] + in - n;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (tie(v[e], at + e)) {
                if ((unsigned long long)before == keep) sh.found[2] = (unsigned long long)(at + e);
                ++before;
            }
        }
    }
    __syncthreads();
    cut.idx = (int)sh.found[2];
}

// The first n of the list sorted, largest first: up to 256 by counting those above each, threads side by side over parts of
// the list; more by a bitonic sort, an element a thread, whose exchanges within a wave need no barrier (four rows of 997
// with top_p 0.9: 22 us, 48 by counting, 26 with every exchange through LDS)
__device__ __forceinline__ void sort_list(Shared& sh, int n) {
    const int tid = threadIdx.x;
    if (n <= 256) {
        int* rank = (int*)sh.bin;
        int len = 64;
        while (len < n) len <<= 1;
        const int i = tid & (len - 1), parts = kThreads / len, per = ceil_div(n, parts), j0 = tid / len * per, j1 = min(j0 + per, n);
        if (tid < len) rank[tid] = 0;
        const unsigned long long mine = i < n ? sh.list[i] : 0;
        __syncthreads();
        int above = 0;
#pragma unroll 4
        for (int j = j0; j < j1; ++j) above += sh.list[j] > mine;
        if (above) atomicAdd(&rank[i], above);
        __syncthreads();
        const int at = i < n && tid < len ? rank[i] : -1;
        if (at >= 0) sh.list[at] = mine;
    } else if (n <= kThreads) {
        unsigned long long x = tid < n ? sh.list[tid] : 0;
        for (int size = 2; size <= kThreads; size <<= 1)
            for (int d = size >> 1; d > 0; d >>= 1) {
                unsigned long long y;
                if (d >= 64) {
                    __syncthreads();
                    sh.list[tid] = x;
                    __syncthreads();
                    y = sh.list[tid ^ d];
                } else {
                    y = __shfl_xor(x, d);
                }
                const bool larger = ((tid & d) == 0) == ((tid & size) == 0);
                if ((y > x) == larger) x = y;
            }
        __syncthreads();
        sh.list[tid] = x;
    } else {
        for (int i = n + tid; i < kList; i += kThreads) sh.list[i] = 0;
        for (int size = 2; size <= kList; size <<= 1)
            for (int d = size >> 1; d > 0; d >>= 1) {
                __syncthreads();
                const int a = ((tid & ~(d - 1)) << 1) | (tid & (d - 1)), b = a | d;
                const unsigned long long x = sh.list[a], y = sh.list[b];
                if ((x < y) == ((a & size) == 0)) {
                    sh.list[a] = y;
                    sh.list[b] = x;
                }
            }
    }
}

// The filters on a list: the elements of keys `least` and more are listed, sorted and cut to the first k and to top_p of
// `whole` (0: of those k).  On return sh.bin holds the kept weights a chunk.  False where the list is too short for them,
// or top_p of `whole` not in it.
template <typename T>
__device__ __forceinline__ bool cut_list(Shared& sh, const Row<T>& row, Cut& cut, uint32_t least, int k, float top_p, unsigned long long least_w,
                                         unsigned long long whole) {
    constexpr int VEC = Row<T>::VEC, PER = kList / kThreads;
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const float low = row.value(least);
    row.seek(sh.top, low, [&](int, int at, const float* v) {
        float m = v[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) m = fmaxf(m, v[e]);
        if (m >= low) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (v[e] >= low) {  // (NaN and absent elements are not)
                    const int o = atomicAdd(&sh.count, 1);
                    if (o < kList) sh.list[o] = ((unsigned long long)key_of<T>(v[e]) << 32) | (uint32_t)~(at + e);
                }
        }
    });
    __syncthreads();
    const int n = sh.count;
    if (n > kList) return false;
    sort_list(sh, n);
    clear_bins(sh, row.chunks);
    const int nk = min(n, k);
    unsigned long long w[PER], sum = 0, total;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int i = tid * PER + e;
        w[e] = i < nk ? row.weight(row.value((uint32_t)(sh.list[i] >> 32))) : 0;
        sum += w[e];
    }
    unsigned long long before = block_scan(sh, sum, total);
    const double thr = (double)top_p * (double)(whole ? whole : total);
    if (whole && (double)total < thr) return false;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int i = tid * PER + e;
        // (what weighs nothing is never drawn, so that it does not matter where it lies to the cut)
        if (i < nk && w[e] >= least_w && w[e] > 0 && (i == 0 || top_p >= 1.f || (double)before < thr)) {
            const int idx = (int)~(uint32_t)sh.list[i];
            atomicAdd(&sh.bin[(idx + row.shift) / Row<T>::CHUNK], w[e]);
            atomicMax(&sh.count, n + 1 + i);
        }
        before += w[e];
    }
    __syncthreads();
    const unsigned long long last = sh.list[sh.count - n - 1];
    cut = {(uint32_t)(last >> 32), (int)~(uint32_t)last + 1};
    return true;
}

// Narrows `cut` to the end of a prefix.  `counts`: the first k elements.  Otherwise those before which less
// than top_p of the weight of `cut` lies (kept as it is if all are).  A histogram over even parts of the weights'
// exponents, over which logits spread as they do over their range, finds the one in which the prefix ends; its elements
// are listed and sorted, or all from there up, where those are few (True: that has cut the row, see cut_list).  Where one
// part holds more than a list does, a radix search goes on over keys.
// (200 float32 rows of 151936, top_p 0.9: 166 us, 270 with a radix search alone, whose first bins few of the logits fill.)
// A call of its own: inlined, the registers it needs cost every row that does without it (float32 rows, temperature
// alone, 75 -> 83 us).  As compiled, a kernel holds 120 vector registers and none of them in scratch, 100 bytes of scratch
// a lane with the call's frame, and 38 (bfloat16: 51) scalar registers spilled.
struct Narrowed {
    Cut cut;
    bool summed;
};

template <typename T>
__device__ __attribute__((noinline)) Narrowed narrow(const Row<T> row, Cut cut, bool counts, unsigned long long k, float top_p,
                                                     unsigned long long least_w) {
    Shared& sh = shared();
    constexpr int VEC = Row<T>::VEC, BITS = Key<T>::bits;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const Cut old = cut;
    unsigned long long above = 0, own = 0, total;  // counted or weighed above the bins searched, in the one found
    double thr = 0;
    uint32_t prefix = 0, bin;
    auto ends = [&](unsigned long long a, unsigned long long h) {
        return counts ? a < k && k <= a + h : (double)a < thr && !((double)(a + h) < thr);
    };
    const float edge = row.value(old.key);
    auto inside = [&](float v, int i) { return old.key == 0 || v > edge || (v == edge && i < old.idx); };
    clear_bins(sh, kBins);
    row.each([&](int, int at, const float* v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const double t = row.exponent(v[e]);
            const int b = row.bin_of(t);
            if (b > 0 && inside(v[e], at + e)) atomicAdd(&sh.bin[b], counts ? 1ull : row.weight_of(t));
        }
    });
    __syncthreads();
    if (!counts) {  // the threshold is a part of the whole
        unsigned long long s = 0;
        for (int b = tid; b < kBins; b += kThreads) s += sh.bin[b];
        block_scan(sh, s, total);
        thr = (double)top_p * (double)total;
        __syncthreads();
    }
    const unsigned long long whole = total;
    if (!find_bin(sh, 12, 0, ends, total, bin, above, own)) return {cut, false};  // everything of weight is kept
    if (counts) {
        if (above + own <= kList && cut_list(sh, row, cut, key_of<T>(row.below_bin((int)bin)), (int)k, top_p, least_w, 0)) return {cut, true};
    } else if (old.key == 0) {
        float n = 0.f;  // elements from that bin up, from their weights: fewer than 1 in 100 off
        for (int b = tid; b < kBins; b += kThreads)
            if (b >= (int)bin) n += (float)sh.bin[b] * exp2f((float)(kBins - 1 - b) * (1.f / (float)kPerUnit) - 42.f);
        block_scan(sh, (unsigned long long)n, total);
        if (total <= kList && cut_list(sh, row, cut, key_of<T>(row.below_bin((int)bin)), row.n, top_p, least_w, whole)) return {cut, true};
    }
    {
        const float lo = row.below_bin((int)bin), hi = row.above_bin((int)bin);
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
        row.seek(sh.top, lo, [&](int, int at, const float* v) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (v[e] >= lo && v[e] <= hi && row.bin_of(row.exponent(v[e])) == (int)bin && inside(v[e], at + e)) {
                    const int o = atomicAdd(&sh.count, 1);
                    if (o < kList) sh.list[o] = ((unsigned long long)key_of<T>(v[e]) << 32) | (uint32_t)~(at + e);
                }
        });
        __syncthreads();
        const int n = sh.count;
        if (n <= kList) {
            sort_list(sh, n);
            __syncthreads();
            int last = (int)(k - above) - 1;
            if (!counts) {
                constexpr int PER = kList / kThreads;
                unsigned long long w[PER], sum = 0;
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int i = tid * PER + e;
                    w[e] = i < n ? row.weight(row.value((uint32_t)(sh.list[i] >> 32))) : 0;
                    sum += w[e];
                }
                unsigned long long before = above + block_scan(sh, sum, total);
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int i = tid * PER + e;
                    if (i < n && (double)before < thr) atomicMax(&sh.count, n + 1 + i);
                    before += w[e];
                }
                __syncthreads();
                last = sh.count - n - 1;
            }
            const unsigned long long x = sh.list[last];
            return {{(uint32_t)(x >> 32), (int)~(uint32_t)x + 1}, false};
        }
    }
    above = 0;
    for (int shift = BITS; shift > 0;) {
        const int width = min(shift, 12), upper = shift;
        shift -= width;
        clear_bins(sh, 1 << width);
        row.each([&](int, int at, const float* v) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const uint32_t kk = key_of<T>(v[e]);
                if ((upper == BITS || (kk >> upper) == prefix) && row.has(at + e) && old.keeps(kk, at + e)) {
                    const unsigned long long w = counts ? 1ull : row.weight(v[e]);
                    if (w) atomicAdd(&sh.bin[(kk >> shift) & ((1u << width) - 1)], w);
                }
            }
        });
        __syncthreads();
        find_bin(sh, width, above, ends, total, bin, above, own);
        prefix = (prefix << width) | bin;
    }
    // equal keys: the first `keep` of them
    unsigned long long keep, ties;
    if (counts) {
        ties = own;
        keep = k - above;
    } else {
        const unsigned long long w = row.weight(row.value(prefix));
        ties = own / w;
        keep = reach(above, w, ties, thr);
    }
    keep_equal(sh, row, cut, prefix, keep, ties);
    return {cut, false};
}

// A key that at least k of the threads' largest keys reach, so at least k elements do: the k-th largest of them, of
// keys over 24 bits to those.  k at most kThreads.
template <int BITS>
__device__ __forceinline__ uint32_t reached_by(Shared& sh, uint32_t mine, unsigned long long k) {
    unsigned long long above = 0, own, total;
    uint32_t prefix = 0;
    int shift = BITS;
    for (int level = 0; level < 2 && shift > 0; ++level) {
        const int width = min(shift, 12), upper = shift;
        shift -= width;
        clear_bins(sh, 1 << width);
        if (upper == BITS || (mine >> upper) == prefix) atomicAdd(&sh.bin[(mine >> shift) & ((1u << width) - 1)], 1ull);
        __syncthreads();
        uint32_t bin;
        find_bin(sh, width, above, [&](unsigned long long a, unsigned long long h) { return a < k && k <= a + h; }, total, bin, above,
                 own);
        prefix = (prefix << width) | bin;
    }
    return prefix << shift;
}

// Weights of bfloat16 logits by value: few values lie between the largest logit and where weights round to 0, so each is
// formed once and an element costs a look-up.  An entry a sign and magnitude (the upper bits of the float32) from a0, the
// second of each sign; the last of each sign stands for all beyond, of weight 0.  Magnitudes below a0 (2^-15 of the largest
// that weighs, and always zeros) have each sign's first entry, of weight 0: they are weighed directly.
// What bounds the passes is the arithmetic of an element, so that entries are found two elements at a time in halves of
// 32 bits, and an entry holds its weight in two parts of 21 bits whose sums over a wave stay below 2^32.
constexpr int kSide = 2048, kTableCols = 16384;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// the entries of a vector of eight logits: within a side, then of the table
struct Entries {
    u16x2 side[4];
    uint32_t two[4];
    __device__ __forceinline__ int operator[](int e) const { return (int)(two[e / 2] >> (e & 1) * 16 & 0xffffu); }
};

struct Table {
    u32x2* w;  // [2 kSide] lower 21 bits, upper bits
    uint32_t a0;

    // the table of a row; weights are 0 below the logit `low`
    __device__ __forceinline__ Table(unsigned long long* lds, const Row<bf16>& row, float low) : w((u32x2*)lds) {
        const float m = (float)row.m;
        const uint32_t up = m > 0.f ? __float_as_uint(m) >> 16 : 0;
        const uint32_t down = low < 0.f ? min((__float_as_uint(-low) >> 16) + 1, 0x7f7fu) : 0;
        const uint32_t most = max(up, down);
        a0 = most > kSide - 3 ? most - (kSide - 3) : 1;
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kSide; i += kThreads) {
            const float v = value(i);
            const unsigned long long x = holds(i) && v <= m ? row.weight(v) : 0;
            w[i] = u32x2{(uint32_t)x & 0x1fffffu, (uint32_t)(x >> 21)};
        }
        __syncthreads();
    }
    __device__ __forceinline__ static bool holds(int i) { return (uint32_t)((i & (kSide - 1)) - 1) < (uint32_t)(kSide - 2); }
    __device__ __forceinline__ unsigned long long weight(int i) const { return ((unsigned long long)w[i][1] << 21) + w[i][0]; }
    __device__ __forceinline__ float value(int i) const {
        return __uint_as_float((uint32_t)(i / kSide) << 31 | ((uint32_t)(i & (kSide - 1)) + a0 - 1) << 16);
    }
    __device__ __forceinline__ Entries entries(u32x4 u) const {
        Entries n;
        const u16x2 less = {(uint16_t)(a0 - 1), (uint16_t)(a0 - 1)}, most = {kSide - 1, kSide - 1};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u16x2 mag = __builtin_bit_cast(u16x2, u[k] & 0x7fff7fffu);
            n.side[k] = __builtin_elementwise_min(__builtin_elementwise_sub_sat(mag, less), most);
            n.two[k] = (u[k] >> 4 & 0x08000800u) | __builtin_bit_cast(uint32_t, n.side[k]);
        }
        return n;
    }
    __device__ __forceinline__ int entry(float v) const {
        return entries(u32x4{__float_as_uint(v) >> 16, 0, 0, 0})[0];
    }
    __device__ __forceinline__ bool in_zone(float v) const { return fabsf(v) < __uint_as_float(a0 << 16); }
    // whether any of eight values is
    __device__ __forceinline__ static bool any_in_zone(const Entries& n) {
        const u16x2 m = __builtin_elementwise_min(__builtin_elementwise_min(n.side[0], n.side[1]),
                                                  __builtin_elementwise_min(n.side[2], n.side[3]));
        return m[0] == 0 || m[1] == 0;
    }
};
__device__ __forceinline__ float element(u32x4 u, int e) { return __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16); }

// The filters from counts of each entry (no list, or more than it holds): `cut` is the last value kept, `keep` how many of it
// (-1: all).  False where a prefix ends among the keys that have no entry.
__device__ __forceinline__ bool cut_table(Shared& sh, const Row<bf16>& row, const Table& tab, Cut& cut, int& keep_out, int top_k, float top_p) {
    constexpr int PER = 2 * kSide / kThreads;
    uint32_t* count = (uint32_t*)sh.list;
    static_assert(2 * kSide * sizeof(uint32_t) <= sizeof(sh.list), "a count an entry");
    unsigned long long* zone = sh.bin;  // elements and weight of the zone
    const int tid = threadIdx.x;
    __syncthreads();
    for (int i = tid; i < 2 * kSide; i += kThreads) count[i] = 0;
    if (tid < 2) zone[tid] = 0;
    __syncthreads();
    row.skim([&](int, int, u32x4 u) {
        const Entries n = tab.entries(u);
        if (tab.any_in_zone(n)) {
#pragma unroll
            for (int e = 0; e < Row<bf16>::VEC; ++e)
                if (tab.in_zone(element(u, e))) {
                    atomicAdd(&zone[0], 1ull);
                    atomicAdd(&zone[1], row.weight(element(u, e)));
                }
        }
#pragma unroll
        for (int e = 0; e < Row<bf16>::VEC; ++e)
            if (n.side[e / 2][e & 1] != kSide - 1) atomicAdd(&count[n[e]], 1u);
    });
    __syncthreads();
    const unsigned long long zn = zone[0], zw = zone[1];
    // a thread's entries from the largest value down, what lies above them, and of how many: positive ones first, then
    // the zone, then negative ones
    auto at = [&](int e) {
        const int r = tid * PER + e;
        return r < kSide ? kSide - 1 - r : r;
    };
    unsigned long long c[PER], w[PER], ca, wa, cn = 0, wn = 0, call, wall;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        c[e] = tab.holds(at(e)) ? count[at(e)] : 0;
        w[e] = tab.weight(at(e));
        cn += c[e];
        wn += c[e] * w[e];
    }
    ca = block_scan(sh, cn, call);
    wa = block_scan(sh, wn, wall);
    call += zn;
    wall += zw;
    auto search = [&](auto ends) {  // the entry in which ends(counted above, weighed above, its count, its weight) holds
        if (tid == 0) sh.found[0] = ~0ull;
        __syncthreads();
        unsigned long long cc = ca, ww = wa;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const bool below = at(e) >= kSide;
            const unsigned long long c0 = cc + (below ? zn : 0), w0 = ww + (below ? zw : 0);
            if (ends(c0, w0, c[e], w[e])) {
                sh.found[0] = (unsigned long long)at(e);
                sh.found[1] = c0;
                sh.found[2] = w0;
                sh.found[3] = c[e];
            }
            cc += c[e];
            ww += c[e] * w[e];
        }
        __syncthreads();
        return sh.found[0] != ~0ull;
    };
    int end = -1;  // the entry that is cut, how many of it are kept, of how many
    unsigned long long keep = 0, ties = 0, whole = wall;
    if (top_k > 0 && (unsigned long long)top_k < call) {
        const unsigned long long k = (unsigned long long)top_k;
        if (!search([&](unsigned long long c0, unsigned long long, unsigned long long n, unsigned long long) { return c0 < k && k <= c0 + n; }))
            return false;
        end = (int)sh.found[0];
        keep = k - sh.found[1];
        ties = sh.found[3];
        whole = sh.found[2] + keep * tab.weight(end);
        __syncthreads();
    }
    if (top_p < 1.f) {
        const double thr = (double)top_p * (double)whole;
        if (search([&](unsigned long long, unsigned long long w0, unsigned long long n, unsigned long long w) {
                return (double)w0 < thr && !((double)(w0 + n * w) < thr);
            })) {
            const int i = (int)sh.found[0];
            const unsigned long long r = reach(sh.found[2], tab.weight(i), sh.found[3], thr);
            keep = i == end && keep < r ? keep : r;
            end = i;
            ties = sh.found[3];
        } else if (!((double)wall < thr)) {
            return false;
        }
        __syncthreads();
    }
    if (end >= 0) {
        cut = {key_of<bf16>(tab.value(end)), 0x7fffffff};
        if (keep < ties) keep_out = (int)keep;
    }
    return true;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
    Shared& sh = shared();
    constexpr int VEC = Row<T>::VEC;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    Row<T> row;
    row.x = (typename Row<T>::global*)p.x + (int64_t)r * p.x_st;
    row.n = p.n_cols;
    row.shift = (int)(((uintptr_t)row.x & 15) / sizeof(T));
    row.chunks = ceil_div(row.n + row.shift, Row<T>::CHUNK);
    const float temp = p.temperature ? p.temperature[r] : p.temperature_all;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_all, min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    const bool filters = (top_k > 0 && top_k < row.n) || top_p < 1.f;
    // the largest logit and the first vector that holds it, and each chunk's largest where chunks may be passed over later
    float best = -INFINITY;
    int best_at = 0;
    float four[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    row.skim(
        [&](int, int at, const float* v) {
            float m = v[0];
#pragma unroll
            for (int e = 1; e < VEC; ++e) m = fmaxf(m, v[e]);
            best_at = m > best ? at + VEC : best_at;  // (more than 0: a row's first vector may begin before it)
            best = fmaxf(best, m);
            four[0] = four[1], four[1] = four[2], four[2] = four[3], four[3] = m;
        },
        [&](int c) {
            if (!filters) return;
            // (after fewer than four, at the row's end, the first of them is not four[0])
            const int n = min((row.chunks - 1 - c) / kWaves + 1, 4), k = ((lane >> 5) | (lane >> 3 & 2)) - (4 - n);
            const uint16_t key = upper_key(wave_max4(four));
            if ((lane & 15) == 0 && k >= 0) sh.top[c + k * kWaves] = key;
        });
    const uint32_t own = key_of<T>(best);
    unsigned long long first = ((unsigned long long)own << 32) | (uint32_t)~best_at;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const unsigned long long b = __shfl_xor(first, o);
        first = b > first ? b : first;
    }
    if (lane == 0) sh.part[wv] = first;
    __syncthreads();
    for (int k = 0; k < kWaves; ++k) first = sh.part[k] > first ? sh.part[k] : first;
    const uint32_t top = __builtin_amdgcn_readfirstlane((uint32_t)(first >> 32));
    const int top_at = (int)~(uint32_t)first - VEC;  // where the vector of the first such logit begins
    if (top == key_of<T>(-INFINITY)) {  // nothing to draw
        if (tid == 0) {
            p.token[r] = -1;
            p.logp[r] = -INFINITY;
        }
        return;
    }
    // the first token alone: greedy, or filters that leave no more (min_p above 1 and NaN among them)
    if (!(temp > 0.f) || top_k == 1 || !(top_p > 0.f) || !(min_p <= 1.f)) {
        if (tid == 0) {
            float v[VEC];
            row.load(top_at, v);
            int top_i = top_at;
#pragma unroll
            for (int e = VEC - 1; e >= 0; --e) top_i = v[e] == row.value(top) ? top_at + e : top_i;
            p.token[r] = top_i;
            p.logp[r] = 0.f;
        }
        return;
    }
    const bool inf = row.value(top) == INFINITY;
    row.m = inf ? 1e39 : (double)row.value(top);
    row.rate = inf ? 1.0 : 1.4426950408889634 / (double)temp;
    const unsigned long long least_w = min_p > 0.f ? (unsigned long long)ceil((double)min_p * (double)kUnit) : 0;
    Cut cut = {0u, 0};
    bool summed = false;
    if (filters && (row.n <= kList || (top_k > 0 && top_k <= kThreads))) {
        uint32_t least = key_of<T>(-INFINITY);
        if (top_k > 0 && top_k <= kThreads) least = max(least, reached_by<Key<T>::bits>(sh, own, (unsigned long long)top_k));
        summed = cut_list(sh, row, cut, least, top_k > 0 ? top_k : row.n, top_p, least_w, 0);
    }
    // kept weights a chunk, then the chunk, lane and element in which the running sum passes u times the total
    const int per = ceil_div(row.chunks, kThreads), c0 = min(tid * per, row.chunks), c1 = min(c0 + per, row.chunks);
    unsigned long long total;
    uint32_t* ties = (uint32_t*)sh.list;  // equal elements at the end of a prefix, a chunk: there, then kept
    bool tied = false;
    if constexpr (Key<T>::bits == 16) {
        // (one row, temperature alone: 8192 12.0 us, 13.1 with a table, 16384 14.0 and 13.5, 32000 18.7 and 15.7; filtered rows
        // past a list's length: 2500 with top_p 0.9 36 and 21)
        if (!summed && (filters || row.n >= kTableCols) && !inf) {
            const Table tab(sample_lds + sizeof(Shared) / sizeof(unsigned long long), row, row.value(top) - 30.f * temp);
            int keep = -1;
            summed = !filters || cut_table(sh, row, tab, cut, keep, top_k, top_p);
            if (summed) {
                // what is not kept weighs nothing from here on, nor does what ends the prefix where it is kept in part: a
                // chunk's number of those is counted, and which of them are kept follows once all are
                const float edge = cut.key ? row.value(cut.key) : -INFINITY;
                tied = keep >= 0;
                const unsigned long long tie_w = tied ? tab.weight(tab.entry(edge)) : 0;
                __syncthreads();
                if (cut.key || least_w)
                    for (int i = tid; i < 2 * kSide; i += kThreads) {
                        const float v = tab.value(i);
                        if (v < edge || (tied && v == edge) || tab.weight(i) < least_w) tab.w[i] = u32x2{0, 0};
                    }
                for (int c = tid; c < row.chunks; c += kThreads) sh.bin[c] = ties[c] = 0;
                __syncthreads();
                const uint32_t edge_bits = __float_as_uint(edge) >> 16;
                auto draw = [&](int c, int, u32x4 u) {
                    const Entries n = tab.entries(u);
                    uint32_t lower = 0, upper = 0;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const u32x2 w = tab.w[n[e]];
                        lower += w[0];
                        upper += w[1];
                    }
                    if (tab.any_in_zone(n)) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float v = element(u, e);
                            const unsigned long long w = tab.in_zone(v) && v > edge ? row.weight(v) : 0;
                            if (w >= least_w) {
                                lower += (uint32_t)w & 0x1fffffu;
                                upper += (uint32_t)(w >> 21);
                            }
                        }
                    }
                    if (__any((lower | upper) != 0)) {
                        const unsigned long long s = wave_sum2<21>(lower, upper);
                        if (lane == 0) sh.bin[c] = s;
                    }
                    if (tied) {
                        uint32_t same = 0;
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            same += (uint32_t)__popcll(__ballot((e & 1 ? u[e / 2] >> 16 : u[e / 2] & 0xffffu) == edge_bits));
                        if (lane == 0) ties[c] = same;
                    }
                };
                if (cut.key) row.seek(sh.top, edge, draw);
                else row.skim(draw);
                __syncthreads();
                if (tied) {
                    unsigned long long n = 0;
                    for (int c = c0; c < c1; ++c) n += ties[c];
                    int64_t left = keep - (int64_t)block_scan(sh, n, total);
                    for (int c = c0; c < c1; ++c) {
                        const int there = (int)ties[c], stay = (int)min(max(left, (int64_t)0), (int64_t)there);
                        left -= there;
                        ties[c] = (uint32_t)stay;
                        if (tie_w >= least_w) sh.bin[c] += (unsigned long long)stay * tie_w;
                    }
                }
            }
        }
    }
    auto chunk_scan = [&] {  // what lies before the thread's chunks, and the total
        unsigned long long s = 0;
        for (int c = c0; c < c1; ++c) s += sh.bin[c];
        return block_scan(sh, s, total);
    };
    auto sums = [&](auto of) {  // a sum a chunk
        __syncthreads();
        row.each([&](int c, int at, const float* v) {
            unsigned long long s = 0;
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += of(v[e], at + e);
            s = wave_sum_weights(s);
            if (lane == 0) sh.bin[c] = s;
        });
        __syncthreads();
    };
#pragma unroll 1
    for (int by_weight = 0; by_weight < 2 && !summed; ++by_weight)
        if (by_weight ? top_p < 1.f : top_k > 0 && top_k < row.n) {
            const Narrowed o = narrow<T>(row, cut, !by_weight, (unsigned long long)top_k, top_p, least_w);
            cut = o.cut;
            summed = o.summed;
        }
    const float edge = row.value(cut.key);
    auto kept = [&](float v, int i) -> unsigned long long {
        if (cut.key && !(v > edge || (v == edge && i < cut.idx))) return 0;
        const unsigned long long w = row.weight(v);
        return w >= least_w ? w : 0;
    };
    if (!summed) {
        if (cut.key == 0) sums([&](float v, int) {
            const unsigned long long w = row.weight(v);
            return w >= least_w ? w : 0;
        });
        else sums(kept);
    }
    __syncthreads();
    unsigned long long cum = chunk_scan();
    double u = p.u_f64 ? ((const double*)p.u)[r] : (double)((const float*)p.u)[r];
    if (!(u >= 0.0)) u = 0.0;
    double goal = u * (double)total;
    if (!((double)total > goal))  // u >= 1: the last kept token (the float64 below the total)
        goal = __longlong_as_double(__double_as_longlong((double)total) - 1);
    for (int c = c0; c < c1; ++c) {
        const unsigned long long next = cum + sh.bin[c];
        if (!((double)cum > goal) && (double)next > goal) {
            sh.found[0] = c;
            sh.found[1] = cum;
        }
        cum = next;
    }
    __syncthreads();
    if (wv == 0) {
        const int at = row.first((int)sh.found[0]);
        float v[VEC];
        row.load(at, v);
        if (tied) {  // the chunk's first equal element that is not kept
            int n = 0, out = 0x7fffffff;
#pragma unroll
            for (int e = 0; e < VEC; ++e) n += v[e] == edge;
            int in = n;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(in, d);
                if (lane >= d) in += o;
            }
            int before = in - n;
            const int stay = (int)ties[(int)sh.found[0]];
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (v[e] == edge) {
                    if (before == stay) out = at + e;
                    ++before;
                }
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) out = min(out, __shfl_xor(out, o));
            cut.idx = out;
        }
        unsigned long long w[VEC], s = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += w[e] = row.has(at + e) ? kept(v[e], at + e) : 0;
        unsigned long long in = s;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const unsigned long long o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        unsigned long long before = sh.found[1] + in - s, weighs = 0;
        int drawn = -1;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (!((double)before > goal) && (double)(before + w[e]) > goal) {
                drawn = at + e;
                weighs = w[e];
            }
            before += w[e];
        }
        if (drawn >= 0) {  // one lane
            p.token[r] = drawn;
            p.logp[r] = (float)log((double)weighs / (double)total);
        }
    }
}

hipError_t sample_some(const SampleParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.rows);
    switch (p.dtype) {
        case 0: DSALT_LAUNCH("sample", sample_kernel<float>, grid, dim3(kThreads), sizeof(Shared), stream, p); break;
        case 1: {
            const unsigned table = p.n_cols > kList ? 2 * kSide * sizeof(unsigned long long) : 0;
            if (table)
                if (hipError_t e = hipFuncSetAttribute((const void*)sample_kernel<bf16>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                       (int)(sizeof(Shared) + table)))
                    return e;
            DSALT_LAUNCH("sample", sample_kernel<bf16>, grid, dim3(kThreads), sizeof(Shared) + table, stream, p);
            break;
        }
        default: DSALT_LAUNCH("sample", sample_kernel<f16>, grid, dim3(kThreads), sizeof(Shared), stream, p); break;
    }
    return hipGetLastError();
}

}  // namespace

// (rows of a launch: its threads stay below 2^32)
hipError_t sample_launch(const SampleParams& p, hipStream_t stream) {
    constexpr int most = (1 << 22) - 1;
    const size_t esize = p.dtype == 0 ? 4 : 2;
    SampleParams s = p;
    for (int64_t r = 0; r < p.rows; r += s.rows) {
        s.rows = (int)std::min((int64_t)most, p.rows - r);
        s.x = (const char*)p.x + r * p.x_st * (int64_t)esize;
        s.u = (const char*)p.u + r * (p.u_f64 ? 8 : 4);
        s.temperature = p.temperature ? p.temperature + r : nullptr;
        s.top_p = p.top_p ? p.top_p + r : nullptr;
        s.min_p = p.min_p ? p.min_p + r : nullptr;
        s.top_k = p.top_k ? p.top_k + r : nullptr;
        s.token = p.token + r;
        s.logp = p.logp + r;
        if (hipError_t e = sample_some(s, stream)) return e;
    }
    return hipSuccess;
}

}  // namespace dsalt
