// Attention of query tokens over the paged 4-bit cache: row t is the token at position pos[t] of request req[t] and
// attends A(i) = [i - w + 1, i] U {landmarks p of its head's set : 0 <= p < i - w + 1}.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j + b_j - m): one pass with a running maximum m and sum.  A
// step takes 32 keys: their codes become bfloat16 operands with the scales taken in (exact), and both products run on the
// matrix cores, with up to 16 columns of queries.  Columns of a window are the query heads that share a key/value head, of
// one row or of rows of one request side by side (drafted tokens); columns of a head's landmarks, which are its own, are those rows.
// Scores, weights and sums are kept in 32 bits.  A key's share of a query is read once for the columns that share it: at 256
// requests (16 query heads on 2, windows of 512, 128 landmarks a head) 93 MB, most of them landmarks, each head its own.
//
// A block has four waves, each with every fourth step of the window and then parts of the landmarks; their maxima, sums and
// values meet in LDS (the windows' pairwise, which leaves room for a second block where there are sixteen columns of 128).  What
// bounds it is the chain of a step, codes to operands, product, maximum, exponents, product, with two waves a SIMD to hide it
// behind (142 to 226 registers a lane, 57 to 63 scalar ones held in vector registers; three waves would spill vector ones, 45 us for
// the 32 us of the 256 requests; eight waves a block 42 us): vector instructions take 0.39 to 0.41 of the cycles, matrix ones 0.07 to 0.18.
// Four fifths of the steps of the 256 requests are landmarks', with one live column of sixteen.  The memory does not bound it: landmarks
// read from the caches save 3 of 37 us there.  With few rows it is
// dependent reads: position, table, tokens, and for landmarks position, table, token.  So the tokens of a step are in registers two
// steps ahead, a wave's landmarks are looked up while its window is read, and numbers of the whole wave (step, page, head) stay in
// scalar registers.  Values pass through LDS as bfloat16 rows, from where the matrix operand is read transposed.
// One request (windows of 512): 12.1 us; 256: 33.8; 64 requests of five rows in float16, 16 heads of 64 on 4: 19.0 us; four requests
// with windows of 131072: 42 us, 143 MB at 3.4 TB/s, 4 us of it the join of the splits.
#include <algorithm>

#include "cache4.h"
#include "common.h"
#include "decode_attn.h"
#include "fp4.h"
#include "tiles.h"
#include "timing.h"

namespace dsalt {

namespace {

constexpr int kStep = 32;  // keys of a step
constexpr int kWaves = 4;  // of a block
constexpr int kParts = 2;  // that their windows are left in: waves kParts and up first, the others join theirs
constexpr uint32_t kNone = 0xffffffffu;

struct AttnPlan {
    int nh, tiles;      // heads of a block, blocks of a key/value head's query heads
    int nr, run_tiles;  // rows of a block, blocks of a request's rows
    int ns, nl;         // splits of a row's window, and of its landmark slots
    int chunk_log;      // a head's landmark slots are 2^chunk_log parts within a block (-1: there are none)
    int kc, kr_log;     // slots of a part, and of a part with what fills it up to a power of two
    int slots, fields;  // slots that a wave looks up at a time, and numbers it keeps of each
    int col_mul;        // c / nh = c col_mul >> 16 for columns c
    __host__ __device__ int chunks() const { return chunk_log < 0 ? 0 : 1 << chunk_log; }
};

// Eight floats as PARTS bfloat16 operands that sum to them: three leave nothing of a float32 (8 bits each), two nothing of a
// float16.  All but the last part are cut off rather than rounded, moves of bytes in place of conversions (a call 1 to 3 % shorter).
template <int PARTS>
__device__ __forceinline__ void cut8(const float* x, bf16x8* o) {
    typedef bf16 pair __attribute__((ext_vector_type(2)));
    typedef float floats __attribute__((ext_vector_type(2)));
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
        u32x4 u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (k + 1 < PARTS) {
                const uint32_t a = __float_as_uint(r[2 * e]), b = __float_as_uint(r[2 * e + 1]);
                u[e] = __builtin_amdgcn_perm(b, a, 0x07060302u);  // the upper halves
                r[2 * e] -= __uint_as_float(a & 0xffff0000u);
                r[2 * e + 1] -= __uint_as_float(b & 0xffff0000u);
            } else {
                u[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((floats{r[2 * e], r[2 * e + 1]}), pair));
            }
        }
        o[k] = __builtin_bit_cast(bf16x8, u);
    }
}

template <typename T, int D>
struct Step {  // one wave's running maximum, sum and weighted values of 16 columns
    // Weights keep all 24 bits for 16-bit outputs too: with two parts up to 2^-16 of each is lost, and 2 to 4 in a thousand bfloat16
    // outputs (16 of float16) are not the exact result's rounding, with three 0.2 to 0.6 (and 1); a call is 2 to 5 % longer.
    static constexpr int QP = Parts<T>::q, PP = 3, KS = D / 32, JN = D / 16, DL = D / 4, KW = DL / 8;
    typedef uint32_t kword __attribute__((ext_vector_type(KW)));
    struct Tokens {  // lane (row16, kg): elements kg DL ... of tokens 16 half + row16, and their scales
        kword key[2], value[2];
        uint32_t key_scale[2], value_scale[2];
    };
    // a wave's values of a step in LDS: bfloat16 rows of a token each
    static constexpr int VROW = D + 16, STAGE = kStep * VROW * 2;
    bf16x8 qf[KS][QP];
    floatx4 acc[JN];
    float m, l;
    uint32_t poison;  // blocks of 32 elements of column row16 that a value which is not finite has reached

    // the lane's query: column row16, elements kg DL + 8 s + e of step s
    __device__ __forceinline__ void begin(const T* q, int kg) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8];
            load8(q + kg * DL + 8 * s, x);
            cut8<QP>(x, qf[s]);
        }
#pragma unroll
        for (int j = 0; j < JN; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.f;
        poison = 0;
    }
    // a token's share of the lane, from the token's first bytes
    __device__ __forceinline__ static void load(const uint8_t* kv, const uint8_t* sc, int kg, int half, Tokens& t) {
        t.key[half] = *(const kword*)(kv + kg * (DL / 2));
        t.value[half] = *(const kword*)(kv + D / 2 + kg * (DL / 2));
        t.key_scale[half] = sc[kg * DL / 32];
        t.value_scale[half] = sc[D / 32 + kg * DL / 32];
    }
    // Values are held apart from those that are NaN: nan[half] has a bit for each lane's, which are staged as zeros.
    __device__ __forceinline__ static bool stage_values(bf16* lds, int row16, int kg, Tokens& t, unsigned long long* nan) {
#pragma unroll
        for (int half = 0; half < 2; ++half) nan[half] = __ballot(t.value_scale[half] == 255u);
        const bool any = __builtin_expect((nan[0] | nan[1]) != 0, 0);
        if (any) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (t.value_scale[half] == 255u) t.value_scale[half] = 127u, t.value[half] = kword{};
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float scale = e8m0(t.value_scale[half]);
#pragma unroll
            for (int i = 0; i < KW; ++i)
                *(bf16x8*)(lds + (half * 16 + row16) * VROW + kg * DL + 8 * i) = e2m1_op(t.value[half][i], scale);
        }
        return any;
    }
    // scores of keys 16 half + 4 kg + r for column row16
    __device__ __forceinline__ void scores(const Tokens& t, float* x) const {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            floatx4 sc = {0.f, 0.f, 0.f, 0.f};
            const float scale = e8m0(t.key_scale[half]);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const bf16x8 kf = e2m1_op(t.key[half][s], scale);
#pragma unroll
                for (int i = 0; i < QP; ++i) sc = mma(kf, qf[s][i], sc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[4 * half + r] = sc[r];
        }
    }
    // The step's scores in base 2 (-inf: masked) and its staged values.  Columns share the matrix operand of the values but not
    // the keys they attend: a value held as NaN (`any`, seldom) is noted for the columns that attend it.
    __device__ __forceinline__ void take(const bf16* lds, int lane, bool any, const unsigned long long* nan, float* x) {
        if (any) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t blocks = 0;
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
                    blocks |= (uint32_t)(nan[e / 4] >> (c * (32 / DL) * 16 + 4 * (lane >> 4) + e % 4)) & 1u ? 1u << c : 0u;
                if (!(x[e] == -INFINITY)) poison |= blocks;
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
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = exp2_(x[e] - mb);
            l += x[e];
        }
        bf16x8 pf[PP];
        cut8<PP>(x, pf);
#pragma unroll
        for (int j = 0; j < JN; ++j) {
            const bf16x8 vf = tr_op16(lds, VROW, 16 * j, 0, lane);
#pragma unroll
            for (int i = 0; i < PP; ++i) acc[j] = mma(vf, pf[i], acc[j]);
        }
    }
    // a part that `end` left, taken in
    __device__ __forceinline__ void join(const float2* ml, const float* out, int kg) {
        const float2 o = *ml;
        if (o.y == 0.f) return;  // (it attended nothing and left no values)
        const float m1 = fmaxf(m, o.x), mb = m1 == -INFINITY ? 0.f : m1;
        const float f = m == -INFINITY ? 1.f : exp2_(m - mb), fo = o.x == -INFINITY ? 1.f : exp2_(o.x - mb);
        m = m1;
        l = l * f + (kg == 0 ? o.y * fo : 0.f);
#pragma unroll
        for (int j = 0; j < JN; ++j) acc[j] = acc[j] * f + *(const floatx4*)(out + 16 * j + 4 * kg) * fo;
    }
    // the wave's part of column row16: (maximum, sum) and, where it took any keys, the weighted values [D]
    __device__ __forceinline__ void end(float2* ml, float* out, int kg, bool column, bool any) {
        const float sum = sum_g4(l);
        const uint32_t all = poison | __shfl_xor(poison, 16);
        const uint32_t nan = all | __shfl_xor(all, 32);
        if (!column) return;
        if (kg == 0) *ml = make_float2(m, sum);
        if (any) {
#pragma unroll
            for (int j = 0; j < JN; ++j) *(floatx4*)(out + 16 * j + 4 * kg) = nan >> (j / 2) & 1u ? floatx4{} + NAN : acc[j];
        }
    }
};

// The parts of a block's columns joined (ml and accs [part][stride columns]; column c is head h0 + c % nh, below h1, of row
// t0 + c / nh): written out, or to the workspace where the row is split.  A part with sum 0 attended nothing and left no values.
template <typename T, int D>
__device__ __forceinline__ void join_columns(const Cache4AttnParams& p, const AttnPlan& a, float2* ml, const float* accs, int parts, int stride,
                                             int cols, int t0, int h0, int h1, int split) {
    float2* total = ml + parts * stride;  // maximum and sum of each column
    const int ns = a.ns;
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += 64 * kWaves) {
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
    for (int i = threadIdx.x; i < cols * D; i += 64 * kWaves) {
        const int c = i / D, d = i - c * D, row = c * a.col_mul >> 16, h = h0 + c - row * a.nh;
        if (h >= h1) continue;
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

// x as a number that the compiler knows nothing of: what is formed from it stays where it is used, where it would otherwise be
// formed ahead of every loop and held in registers through all of them
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

constexpr int kLook = 4;  // slots that a lane looks up at a time, at most

// LDS of a block: (maximum, sum) and weighted values of each part and column, the columns' queries, and of each wave the
// keys of its landmarks (page, head and token in one number; kNone: not attended), their positions and biases in base 2, and
// the tokens of its step
template <typename T, int D>
struct Layout {
    static constexpr int QS = D + 16 / (int)sizeof(T);  // a query's elements and what keeps rows apart in the banks
    int parts, stride, wave_slots;
    __host__ __device__ Layout(const AttnPlan& a) : parts(kParts + a.chunks()), stride(a.nr * a.nh), wave_slots(a.slots * a.fields) {}
    __host__ __device__ int ml() const { return 0; }
    __host__ __device__ int q() const { return (2 * (parts + 1) * stride + 3) / 4 * 16; }
    __host__ __device__ int slots() const { return q() + stride * QS * (int)sizeof(T); }
    __host__ __device__ int stage() const { return slots() + kWaves * wave_slots * 4; }
    __host__ __device__ int accs() const { return stage() + kWaves * Step<T, D>::STAGE; }
    __host__ __device__ int bytes() const { return accs() + parts * stride * D * 4; }
};

// A block takes rows of one request, side by side, and query heads of one key/value head, 16 columns at most: their
// window, then each head's landmarks.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void cache4_attn_kernel(Cache4AttnParams p, AttnPlan a) {
    typedef Step<T, D> S;
    constexpr int QS = Layout<T, D>::QS;
    extern __shared__ char lds[];
    const Layout<T, D> at(a);
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int G = p.c.n_kv, group = p.n_heads / G, bt_log = p.c.bt_log, bt = 1 << bt_log;
    const int rt = xcd_swizzle(blockIdx.x, gridDim.x), split = blockIdx.z;
    const int g = a.tiles == 1 ? blockIdx.y : blockIdx.y / a.tiles, hx = blockIdx.y - g * a.tiles;
    const int h0 = g * group + hx * a.nh, h1 = min(h0 + a.nh, (g + 1) * group), nh = a.nh;
    const bool marks = split < a.nl;
    const int parts = kParts + (marks ? a.chunks() : 0), stride = at.stride;
    float2* ml = (float2*)(lds + at.ml());
    float* accs = (float*)(lds + at.accs());
    T* qs = (T*)(lds + at.q());
    uint32_t* keys = (uint32_t*)(lds + at.slots()) + wv * at.wave_slots;
    int* places = (int*)keys + (a.nr > 1 ? a.slots : 0);  // (where there are several rows)
    float* biases = (float*)places + a.slots;             // (where there are any)
    bf16* stage = (bf16*)(lds + at.stage() + wv * S::STAGE);
    const float scale2 = p.scale * kLog2e;
    const int run = a.run_tiles == 1 ? rt : rt / a.run_tiles;
    const int64_t t_first = (int64_t)run * p.per + (int64_t)(rt - run * a.run_tiles) * a.nr;
    const int64_t t_end = min(min(t_first + a.nr, ((int64_t)run + 1) * p.per), (int64_t)p.n_rows);
    auto row_of = [&](int c) { return c * a.col_mul >> 16; };
    // the tile's rows, a lane each
    int rq = -1, ps = -1, wd = 1;
    {
        const int64_t t = t_first + (threadIdx.x & 15);
        if (t < t_end) {
            rq = p.req[t];
            ps = p.pos[t];
            wd = max(p.w[t], 1);
        }
    }
    S s;

    for (int64_t tt = t_first; tt < t_end;) {  // (once, unless the rows side by side belong to several requests)
        const int tid = fresh(threadIdx.x), lane = tid & 63, row16 = lane & 15, kg = lane >> 4;
        const int t0 = (int)tt, r0 = (int)(tt - t_first), req = __builtin_amdgcn_readlane(rq, r0);
        const uint32_t others = (((uint32_t)__ballot(rq != req || t_first + row16 >= t_end) & 0xffffu) | 0x10000u) >> r0;
        const int n = __builtin_ctz(others);
        tt += n;
        const int cols = n * nh;
        const bool known = req >= 0 && req < p.n_reqs;
        const int32_t* table = p.table + (known ? (int64_t)req * p.table_st : 0);
        const int cap = (p.cols << bt_log) - 1;
        // rows: the lane's for columns of the window, and for those of landmarks
        struct Range { int low, end; };  // first and last key of the window; a row without keys sees nothing
        auto range = [&](int row) {
            const int pos = __shfl(ps, r0 + row), w = __shfl(wd, r0 + row);
            const bool live = known && pos >= 0;
            return Range{live ? max(pos - w + 1, 0) : 0x7fffffff, live ? min(pos, cap) : -1};
        };
        const int col = row16 < cols ? row16 : 0, lrow = row16 < n ? row16 : 0;
        const Range win = range(row_of(col));
        const int low_r = n == 1 ? win.low : range(lrow).low, mark_low = low_r == 0x7fffffff ? 0 : low_r;
        auto lowest = [](int v) { return __builtin_amdgcn_readfirstlane(row_min16(v)); };
        auto largest = [](int v) { return __builtin_amdgcn_readfirstlane(row_max16(v)); };
        const int low_min = lowest(win.low), low_max = largest(win.low), end_min = lowest(win.end), end_max = largest(win.end);
        const int mark_max = largest(mark_low);

        // ---- the wave's landmarks: slot f of its items (head, part), one after the other
        const int items = marks ? (h1 - h0) << a.chunk_log : 0, my_items = wv < items ? (items - 1 - wv) / kWaves + 1 : 0;
        const int total = known ? my_items << a.kr_log : 0, k0 = split * (a.kc << max(a.chunk_log, 0));
        int mj[kLook];
        float mb[kLook];
        auto look_marks = [&](int b) {
#pragma unroll
            for (int i = 0; i < kLook; ++i) {
                mj[i] = -1;
                mb[i] = 0.f;
                if (i * 64 >= a.slots || b + i * 64 >= total) continue;
                const int f = b + i * 64 + lane, it = wv + (f >> a.kr_log) * kWaves, hh = it >> a.chunk_log;
                const int o = f & ((1 << a.kr_log) - 1), k = k0 + (it - (hh << a.chunk_log)) * a.kc + o;
                if (f < total && o < a.kc && k < p.k_lmk) {
                    const int64_t x = ((int64_t)(h0 + hh) * p.n_reqs + req) * p.k_lmk + k;
                    mj[i] = p.lmk[x];
                    if (p.lbias) mb[i] = p.lbias[x];
                }
            }
        };
        auto place_marks = [&](int b) {  // (after look_marks; a bias of minus infinity masks its key, which is then not read)
            int page[kLook];
#pragma unroll
            for (int i = 0; i < kLook; ++i) {
                const int pb = mj[i] >> bt_log;
                page[i] = -1;
                if (mj[i] >= 0 && mj[i] < mark_max && pb < p.cols && mb[i] != -INFINITY) page[i] = table[pb];
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < kLook; ++i) {
                if (i * 64 >= a.slots || b + i * 64 >= total) continue;
                const bool ok = page[i] >= 0 && page[i] < p.c.n_blocks;
                keys[i * 64 + lane] = ok ? (((uint32_t)page[i] * (uint32_t)G + (uint32_t)g) << bt_log) + (uint32_t)(mj[i] & (bt - 1)) : kNone;
                if (n > 1) places[i * 64 + lane] = mj[i];
                // (the type's lowest values stay finite, as masks of them are apart from minus infinity)
                if (p.lbias) biases[i * 64 + lane] = mb[i] > -INFINITY ? fmaxf(mb[i] * kLog2e, -3e38f) : mb[i];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };

        // ---- window: keys base + 32 step ..., from the aligned position at or before the first
        const int base = low_min & ~(kStep - 1);
        const int steps = end_max >= low_min ? ((end_max - base) >> 5) + 1 : 0, per = a.ns == 1 ? steps : ceil_div(steps, a.ns);
        const int s0 = split * per, s1 = min(steps, s0 + per);
        const int first = s0 + wv, mine = first < s1 ? (s1 - 1 - first) / kWaves + 1 : 0;
        // lane 2 i + half: page (-1: none) of the 16 keys `half` of step i of the batch of 32 steps from b0
        auto look = [&](int b0) {
            const int b = (base + (first + (b0 + (lane >> 1)) * kWaves) * kStep + (lane & 1) * 16) >> bt_log;
            const bool in = b0 + (lane >> 1) < mine && b < p.cols;
            const int page = table[in ? b : 0];
            return in && page >= 0 && page < p.c.n_blocks ? page : -1;
        };
        int page = mine > 0 ? look(0) : -1;
        look_marks(0);
        {  // the columns' queries; parts of landmarks that no item writes hold nothing
            constexpr int VEC = 16 / (int)sizeof(T);
            for (int i = tid; i < cols * (D / VEC); i += 64 * kWaves) {
                const int c = i / (D / VEC), e = i - c * (D / VEC), row = row_of(c), h = min(h0 + c - row * nh, h1 - 1);
                *(u32x4*)(qs + c * QS + e * VEC) =
                    *(const u32x4*)((const T*)p.q + (int64_t)(t0 + row) * p.q_st + (int64_t)h * p.q_sh + e * VEC);
            }
            for (int i = tid; i < (parts - kParts) * stride; i += 64 * kWaves) ml[kParts * stride + i] = make_float2(-INFINITY, 0.f);
        }
        // Tokens of a step, requested two steps ahead: memory answers later than one step takes.
        typename S::Tokens tk[2];
        {
            int held[2] = {0, 0};  // whether the table names the pages of a step's halves
            auto load = [&](int i, typename S::Tokens& t, int& on) {
                if ((i & 31) == 0 && i > 0) page = look(i);
                on = 0;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int pg = __builtin_amdgcn_readlane(page, 2 * (i & 31) + half);
                    on |= pg >= 0 ? 1 << half : 0;
                    const int j = base + (first + i * kWaves) * kStep + half * 16;  // (page 0 where there is none)
                    const uint64_t token = (((uint64_t)max(pg, 0) * G + g) << bt_log) + (j & (bt - 1));
                    S::load(p.c.kv + token * D + row16 * D, p.c.scale + token * (D / 16) + row16 * (D / 16), kg, half, t);
                }
            };
            if (mine > 0) load(0, tk[0], held[0]);
            if (mine > 1) load(1, tk[1], held[1]);
            if (total > 0) place_marks(0);
            __syncthreads();
            s.begin(qs + col * QS, kg);
            auto step = [&](int i, typename S::Tokens& t, int& on) {
                const int j0 = base + (first + i * kWaves) * kStep, both = on;
                float x[8];
                unsigned long long nan[2];
                s.scores(t, x);
                const bool any = S::stage_values(stage, row16, kg, t, nan);
                if (i + 2 < mine) load(i + 2, t, on);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= scale2;
                if (!(j0 >= low_max && j0 + kStep - 1 <= end_min && both == 3)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int j = j0 + (e & 4) * 4 + 4 * kg + (e & 3);
                        const bool out = (j < win.low) | (j > win.end) | !(both >> e / 4 & 1);
                        x[e] = out ? -INFINITY : x[e];
                    }
                }
                s.take(stage, lane, any, nan, x);
            };
#pragma unroll 1
            for (int i = 0; i < mine; i += 2) {
                step(i, tk[0], held[0]);
                if (i + 1 < mine) step(i + 1, tk[1], held[1]);
            }
            // (a wave has steps wherever a later one has)
            const int slot = (wv & (kParts - 1)) * stride + row16;
            if (wv >= kParts) s.end(ml + slot, accs + slot * D, kg, row16 < cols, mine > 0);
            __syncthreads();
            if (wv < kParts) {
                if (row16 < cols) s.join(ml + slot, accs + slot * D, kg);
                s.end(ml + slot, accs + slot * D, kg, row16 < cols, mine > 0);
            }
        }

        // ---- landmarks, whole steps of one item each
        for (int b = 0; b < total; b += a.slots) {
            if (b > 0) {
                look_marks(b);
                place_marks(b);
            }
            const int lane = fresh(threadIdx.x) & 63, row16 = lane & 15, kg = lane >> 4;
            auto load = [&](int i, typename S::Tokens& t) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t key = keys[i * kStep + half * 16 + row16];
                    t.key[half] = t.value[half] = typename S::kword{};
                    t.key_scale[half] = t.value_scale[half] = 127u;
                    if (key != kNone) S::load(p.c.kv + (uint64_t)key * D, p.c.scale + (uint64_t)key * (D / 16), kg, half, t);
                }
            };
            const int n_steps = min(a.slots, total - b) / kStep;
            auto step = [&](int i, typename S::Tokens& t) {
                const int f = b + i * kStep, o = f & ((1 << a.kr_log) - 1), it = wv + (f >> a.kr_log) * kWaves, hh = it >> a.chunk_log;
                if (o == 0) s.begin(qs + (lrow * nh + hh) * QS, kg);
                float x[8];
                unsigned long long nan[2];
                s.scores(t, x);
                const bool any = S::stage_values(stage, row16, kg, t, nan);
                if (i + 2 < n_steps) load(i + 2, t);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int q0 = i * kStep + half * 16 + 4 * kg;
                    const u32x4 key = *(const u32x4*)(keys + q0);
                    u32x4 place = {};
                    if (n > 1) place = *(const u32x4*)(places + q0);
                    floatx4 bias = {};
                    if (p.lbias) bias = *(const floatx4*)(biases + q0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool on = (key[e] != kNone) & ((n == 1) | ((int)place[e] < mark_low));
                        x[4 * half + e] = on ? x[4 * half + e] * scale2 + bias[e] : -INFINITY;
                    }
                }
                s.take(stage, lane, any, nan, x);
                if (o + kStep == 1 << a.kr_log) {
                    const int part = kParts + it - (hh << a.chunk_log), slot = part * stride + row16 * nh + hh;
                    s.end(ml + slot, accs + (int64_t)slot * D, kg, row16 < n, true);
                }
            };
            load(0, tk[0]);
            if (n_steps > 1) load(1, tk[1]);
#pragma unroll 1
            for (int i = 0; i < n_steps; i += 2) {
                step(i, tk[0]);
                if (i + 1 < n_steps) step(i + 1, tk[1]);
            }
        }
        join_columns<T, D>(p, a, ml, accs, parts, stride, cols, t0, h0, h1, split);
        __syncthreads();
    }
}

// How a launch is cut.  The most columns that fit share each key; where that leaves compute units without work, heads go to blocks
// of their own (their landmarks are their own anyhow, and the window's keys are then read from the caches) and long windows to splits.
// Measured, bfloat16, 16 query heads of 128 on 2 with 128 landmarks, us by heads of a block (weights in two parts; three add 2 to 6 %):
//   windows of 512, one row a request: 256 requests 8 heads 33, 4 43; 128: 8 27, 4 24; 64: 8 26, 4 19.5, 2 19.3; 32: 4 18.3, 2 15.4,
//     1 17.6; 8: 2 14.3, 1 13.6; 1: 8 22, 1 11; five rows a request: 256 requests 3 heads 76, 2 82; 64: 3 28, 2 24; 16: 3 22, 2 18,
//     1 16.4.  So heads are halved while that leaves no more than 512 blocks, two a compute unit, which the card holds at once, and to
//     single heads from fewer than 256.
//   sixteen rows of 64 requests, 16 heads of 128: all in a block 51, eight 76, four 128.
//   one request, windows of 4096: 4 heads in 16 splits 16.4, single heads without splits 39.8; 16 requests, 16384: 8 heads in
//     16 splits 32.4; 4 requests, 131072: 48 splits 47, 64 42 (40 since), 96 54, 128 52.  So long windows are split until
//     there are 512 blocks, 256 keys to a split at least, and heads halved only where that is not enough.
AttnPlan attn_plan(const Cache4AttnParams& p) {
    AttnPlan a;
    const int group = p.n_heads / p.c.n_kv;
    const int64_t cap = (int64_t)p.cols << p.c.bt_log;
    const int64_t w = p.w_max > 0 && p.w_max < cap ? p.w_max : cap;
    const int64_t rows = std::max(p.n_rows, 1);  // (the workspace of a call without rows is asked for too)
    a.run_tiles = ceil_div(p.per, 16);
    a.nr = ceil_div(p.per, a.run_tiles);
    a.nh = ceil_div(group, ceil_div(group, 16 / a.nr));
    const int64_t groups = (rows + p.per - 1) / p.per * a.run_tiles * p.c.n_kv;
    auto blocks_of = [&](int nh) { return groups * ceil_div(group, nh); };
    auto blocks = [&] { return blocks_of(a.nh); };
    auto splits = [&](int64_t most) { return std::max(std::min(most / blocks(), w / 256), (int64_t)1); };
    if (w <= 1024) {
        while (a.nh > 1 && blocks_of(ceil_div(a.nh, 2)) <= 512 && (a.nh > 2 || blocks() < 256)) a.nh = ceil_div(a.nh, 2);
        a.ns = w > 512 ? (int)splits(256) : 1;
    } else {
        while (a.nh > 4 && blocks() * splits(512) <= 128) a.nh = ceil_div(a.nh, 2);
        a.ns = (int)splits(512);
    }
    a.tiles = ceil_div(group, a.nh);
    a.nl = p.k_lmk == 0 ? 0 : std::min(ceil_div(p.k_lmk, 32), a.ns);
    a.chunk_log = p.k_lmk == 0 ? -1 : 0;
    if (p.k_lmk > 0)  // (no more parts than leave room for two blocks in a compute unit's LDS: sixteen columns of 128 with four 51 us,
                      // three 53, a block alone 88; float32 rows in pairs with biases, eight heads a block, pass it by 768 bytes)
        while ((2 << a.chunk_log) * a.nh <= kWaves && (kParts + (2 << a.chunk_log)) * a.nr * a.nh * p.c.head_dim * 4 <= 1 << 15) ++a.chunk_log;
    a.kc = p.k_lmk == 0 ? 0 : ceil_div(ceil_div(p.k_lmk, a.nl), a.chunks());
    a.kr_log = 5;
    while (1 << a.kr_log < a.kc) ++a.kr_log;
    a.slots = p.k_lmk == 0 ? 0 : std::min((ceil_div(a.nh << a.chunk_log, kWaves) << a.kr_log) + 63 & ~63, 64 * kLook);
    a.fields = 1 + (a.nr > 1) + (p.lbias != nullptr);
    a.col_mul = ceil_div(1 << 16, a.nh);
    return a;
}

template <typename T, int D>
hipError_t run_rows(const Cache4AttnParams& p, const AttnPlan& a, hipStream_t stream) {
    const int64_t runs = ((int64_t)p.n_rows + p.per - 1) / p.per;
    const dim3 grid((unsigned)(runs * a.run_tiles), (unsigned)(p.c.n_kv * a.tiles), (unsigned)a.ns);
    const unsigned lds = (unsigned)Layout<T, D>(a).bytes();
    auto kernel = cache4_attn_kernel<T, D>;
    if (lds > 65536)
        if (hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)) return e;
    DSALT_LAUNCH("cache4_attn", kernel, grid, dim3(64 * kWaves), lds, stream, p, a);
    if (a.ns > 1) {
        const dim3 join((unsigned)((int64_t)p.n_rows * p.n_heads));
        DSALT_LAUNCH("cache4_attn_join", (cache_attn_join_kernel<T, D, Cache4AttnParams>), join, dim3(64 * kJoinWaves), 0, stream, p, a.ns);
    }
    return hipGetLastError();
}

template <typename T, int D>
hipError_t run(const Cache4AttnParams& p, hipStream_t stream) {
    const AttnPlan a = attn_plan(p);
    // runs of rows of a launch (where there is more than one launch, rows are not split)
    const int64_t most = std::max(kLaunchThreads / 256 / a.run_tiles, (int64_t)1) * p.per;
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
