// One token a row of logits, drawn from given random numbers u in [0, 1).
//
// Order the row's tokens by logit, largest first, equal ones by index.  With m the largest logit, a token
// weighs round(2^42 exp((x - m) / temperature)), a whole number: sums of weights do not depend on their
// order, so that a draw is the same whatever the blocks and lanes that form them.  Kept is a prefix of the
// order: the first top_k tokens, of those the ones before which less than top_p of their weight lies, of
// those the ones that weigh at least min_p 2^42.  The token is the first index whose running sum of kept
// weights, in the order of the vocabulary, passes u times the total.
//
// A block takes a row.  The end of a prefix is found by a radix search over order-preserving keys: a
// histogram (of counts for top_k, of weights for top_p) over twelve bits of the key at a time, the bins
// summed from the top down to the one that holds the end.
#include "common.h"
#include "sample.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 4096;
constexpr double kUnit = 4398046511104.0;  // 2^42: sums over 2^20 tokens stay below 2^62

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
    unsigned long long part[kWaves];
    unsigned long long found[4];
};

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

template <typename T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T), CHUNK = 64 * VEC;
    const T* x;
    int n, shift;  // elements, and those of the first 16-byte vector that lie before the row
    int chunks;
    float m;       // largest logit
    double inv_t;  // 1 / temperature

    // Chunk c: elements c CHUNK - shift ..., VEC a lane from `first`; absent ones get key 0.
    __device__ __forceinline__ int first(int c) const { return c * CHUNK + (int)(threadIdx.x & 63) * VEC - shift; }
    __device__ __forceinline__ void load(int at, float* v) const {
        typedef T vec __attribute__((ext_vector_type(VEC), aligned(16)));
        if (at >= 0 && at + VEC <= n) {
            const vec u = *(const vec*)(x + at);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = to_float(u[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = at + e >= 0 && at + e < n ? to_float(x[at + e]) : 0.f;
        }
    }
    __device__ __forceinline__ uint32_t key(int i, float v) const { return i >= 0 && i < n ? key_of<T>(v) : 0u; }
    __device__ __forceinline__ unsigned long long weight(float v) const {
        if (!(v > -INFINITY)) return 0;
        if (m == INFINITY) return v == m ? (unsigned long long)kUnit : 0;
        return (unsigned long long)rint(exp(((double)v - (double)m) * inv_t) * kUnit);
    }
};

// Narrows `cut` to the end of a prefix.  COUNT: the first k elements.  Otherwise those before which less
// than top_p of the weight of `cut` lies (kept as it is if all are).
template <typename T, bool COUNT>
__device__ void narrow(Shared& sh, const Row<T>& row, Cut& cut, unsigned long long k, float top_p) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const Cut old = cut;
    unsigned long long above = 0;  // counted or weighed above the bins searched
    double thr = 0;
    uint32_t prefix = 0;
    int shift = Key<T>::bits, width = 0;
    while (shift > 0) {
        width = min(shift, 12);
        const int upper = shift;
        shift -= width;
        __syncthreads();
        for (int b = tid; b < (1 << width); b += kThreads) sh.bin[b] = 0;
        __syncthreads();
        for (int c = wv; c < row.chunks; c += kWaves) {
            float v[Row<T>::VEC];
            const int at = row.first(c);
            row.load(at, v);
#pragma unroll
            for (int e = 0; e < Row<T>::VEC; ++e) {
                const uint32_t kk = row.key(at + e, v[e]);
                if (kk != 0 && (upper == Key<T>::bits || (kk >> upper) == prefix) && old.keeps(kk, at + e)) {
                    const unsigned long long w = COUNT ? 1ull : row.weight(v[e]);
                    if (w) atomicAdd(&sh.bin[(kk >> shift) & ((1u << width) - 1)], w);
                }
            }
        }
        __syncthreads();
        // bins from the top: thread t sums those from 4 t on
        const int nb = 1 << width;
        unsigned long long h[4], sum = 0, total;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int b = nb - 1 - (tid * 4 + e);
            h[e] = b >= 0 ? sh.bin[b] : 0;
            sum += h[e];
        }
        unsigned long long cum = above + block_scan(sh, sum, total);
        if (!COUNT && upper == Key<T>::bits) thr = (double)top_p * (double)total;
        if (tid == 0) sh.found[0] = ~0ull;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool ends = COUNT ? cum < k && k <= cum + h[e] : (double)cum < thr && !((double)(cum + h[e]) < thr);
            if (ends) {  // one bin at most
                sh.found[0] = (unsigned long long)(nb - 1 - (tid * 4 + e));
                sh.found[1] = cum;
                sh.found[2] = h[e];
            }
            cum += h[e];
        }
        __syncthreads();
        if (sh.found[0] == ~0ull) return;  // everything is kept
        prefix = (prefix << width) | (uint32_t)sh.found[0];
        above = sh.found[1];
    }
    // equal keys: the first `keep` of them
    const unsigned long long in_bin = sh.found[2];
    unsigned long long keep, ties;
    if (COUNT) {
        ties = in_bin;
        keep = k - above;
    } else {
        const uint32_t full = prefix << (32 - Key<T>::bits);
        const uint32_t u = full >> 31 ? full ^ 0x80000000u : ~(full | (Key<T>::bits < 32 ? (1u << (32 - Key<T>::bits)) - 1 : 0u));
        const unsigned long long w = row.weight(__uint_as_float(u));
        ties = in_bin / w;
        unsigned long long lo = 1, hi = ties;  // the least number after which the weight is reached
        while (lo < hi) {
            const unsigned long long mid = (lo + hi) >> 1;
            if ((double)(above + mid * w) < thr) lo = mid + 1;
            else hi = mid;
        }
        keep = lo;
    }
    cut.key = prefix;
    cut.idx = prefix == old.key ? old.idx : 0x7fffffff;
    if (keep >= ties) return;
    // the index of the first equal key left out
    __syncthreads();
    for (int c = wv; c < row.chunks; c += kWaves) {
        float v[Row<T>::VEC];
        const int at = row.first(c);
        row.load(at, v);
        int n = 0;
#pragma unroll
        for (int e = 0; e < Row<T>::VEC; ++e) n += row.key(at + e, v[e]) == prefix && old.keeps(prefix, at + e);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) n += wave_xor(n, o);
        if (lane == 0) sh.bin[c] = n;
    }
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
        float v[Row<T>::VEC];
        row.load(at, v);
        int n = 0;
#pragma unroll
        for (int e = 0; e < Row<T>::VEC; ++e) n += row.key(at + e, v[e]) == prefix && old.keeps(prefix, at + e);
        int in = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        int before = (int)sh.found[1] + in - n;
#pragma unroll
        for (int e = 0; e < Row<T>::VEC; ++e) {
            if (row.key(at + e, v[e]) == prefix && old.keeps(prefix, at + e)) {
                if ((unsigned long long)before == keep) sh.found[2] = (unsigned long long)(at + e);
                ++before;
            }
        }
    }
    __syncthreads();
    cut.idx = (int)sh.found[2];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
    __shared__ Shared sh;
    constexpr int VEC = Row<T>::VEC;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    Row<T> row;
    row.x = (const T*)p.x + (int64_t)r * p.x_st;
    row.n = p.n_cols;
    row.shift = (int)(((uintptr_t)row.x & 15) / sizeof(T));
    row.chunks = ceil_div(row.n + row.shift, Row<T>::CHUNK);
    const float temp = p.temperature ? p.temperature[r] : p.temperature_all;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_all, min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    // the largest logit and its first index
    unsigned long long best = 0;
    for (int c = wv; c < row.chunks; c += kWaves) {
        float v[VEC];
        const int at = row.first(c);
        row.load(at, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const uint32_t k = row.key(at + e, v[e]);
            const unsigned long long o = ((unsigned long long)k << 32) | (uint32_t)~(at + e);
            if (k && o > best) best = o;
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const unsigned long long b = __shfl_xor(best, o);
        best = b > best ? b : best;
    }
    if (lane == 0) sh.part[wv] = best;
    __syncthreads();
    for (int k = 0; k < kWaves; ++k) best = sh.part[k] > best ? sh.part[k] : best;
    const uint32_t top = (uint32_t)(best >> 32);
    const int top_i = (int)~(uint32_t)best;
    if (top == key_of<T>(-INFINITY)) {  // nothing to draw
        if (tid == 0) {
            p.token[r] = -1;
            p.logp[r] = -INFINITY;
        }
        return;
    }
    if (!(temp > 0.f) || top_k == 1) {
        if (tid == 0) {
            p.token[r] = top_i;
            p.logp[r] = 0.f;
        }
        return;
    }
    row.m = to_float(row.x[top_i]);
    row.inv_t = 1.0 / (double)temp;
    Cut cut = {0u, 0};
    if (top_k > 0 && top_k < row.n) narrow<T, true>(sh, row, cut, (unsigned long long)top_k, 1.f);
    if (!(top_p > 0.f)) cut = {top, top_i + 1};
    else if (top_p < 1.f) narrow<T, false>(sh, row, cut, 0, top_p);
    // kept weights a chunk, then the chunk, lane and element in which the running sum passes u times the total
    const double least = (double)min_p * kUnit;
    auto kept = [&](float v, int i) -> unsigned long long {
        const uint32_t k = row.key(i, v);
        if (k == 0 || !cut.keeps(k, i)) return 0;
        const unsigned long long w = row.weight(v);
        return (double)w >= least || i == top_i ? w : 0;
    };
    __syncthreads();
    for (int c = wv; c < row.chunks; c += kWaves) {
        float v[VEC];
        const int at = row.first(c);
        row.load(at, v);
        unsigned long long s = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += kept(v[e], at + e);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) sh.bin[c] = s;
    }
    __syncthreads();
    const int per = ceil_div(row.chunks, kThreads), c0 = min(tid * per, row.chunks), c1 = min(c0 + per, row.chunks);
    unsigned long long sum = 0, total;
    for (int c = c0; c < c1; ++c) sum += sh.bin[c];
    unsigned long long cum = block_scan(sh, sum, total);
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
        unsigned long long w[VEC], s = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += w[e] = kept(v[e], at + e);
        unsigned long long in = s;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const unsigned long long o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        unsigned long long before = sh.found[1] + in - s;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (!((double)before > goal) && (double)(before + w[e]) > goal) {
                p.token[r] = at + e;
                p.logp[r] = (float)log((double)w[e] / (double)total);
            }
            before += w[e];
        }
    }
}

}  // namespace

hipError_t sample_launch(const SampleParams& p, hipStream_t stream) {
    if (p.rows == 0) return hipSuccess;
    const dim3 grid((unsigned)p.rows);
    switch (p.dtype) {
        case 0: DSALT_LAUNCH("sample", sample_kernel<float>, grid, dim3(kThreads), 0, stream, p); break;
        case 1: DSALT_LAUNCH("sample", sample_kernel<bf16>, grid, dim3(kThreads), 0, stream, p); break;
        default: DSALT_LAUNCH("sample", sample_kernel<f16>, grid, dim3(kThreads), 0, stream, p); break;
    }
    return hipGetLastError();
}

}  // namespace dsalt
