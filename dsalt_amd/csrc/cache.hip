// A decoding step's row maps over a paged cache, and the cache's write and read-back.
#include <algorithm>

#include "cache.h"
#include "common.h"
#include "fp8.h"
#include "timing.h"

namespace dsalt {

namespace {

// ------------------------------------------------------------------ row maps
// Request r holds L tokens in H = ceil(L / b) pages (b tokens a page) and brings n: it needs
// ceil((L + n) / b) - H more.  Prefix sums over the requests, in their order, place its rows, its new
// pages in the ring of free ones, its pieces (runs of rows within one page) and the pages it gives
// back.  One block forms the sums; then a thread a row writes the maps and a wave a request the ring.
struct ReqPlan {
    int32_t state;  // 0 refused, 1 granted, 2 released
    int32_t piece;  // its first piece
    int64_t take;   // its first page among those taken from the ring
    int64_t give;   // its first page among those given back
};

struct Sums {
    int64_t rows, need, give, pieces;
};

__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
    return {a.rows + b.rows, a.need + b.need, a.give + b.give, a.pieces + b.pieces};
}

__device__ __forceinline__ Sums shfl_up(const Sums& s, int d) {
    return {__shfl_up(s.rows, d), __shfl_up(s.need, d), __shfl_up(s.give, d), __shfl_up(s.pieces, d)};
}

constexpr int kPlanThreads = 1024;

// what request r adds, given the rows before it (they decide whether its own fit)
__device__ __forceinline__ int held_pages(const CacheRowsParams& p, int64_t len) {
    return (int)min(max((len + (1 << p.bt_log) - 1) >> p.bt_log, (int64_t)0), (int64_t)p.cols);
}

__global__ __launch_bounds__(kPlanThreads) void rows_plan_kernel(CacheRowsParams p) {
    __shared__ Sums part[kPlanThreads / 64];
    __shared__ int64_t taken_s;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int R = p.n_reqs, bt = 1 << p.bt_log;
    const int per = ceil_div(R, kPlanThreads);
    const int r0 = min(tid * per, R), r1 = min(r0 + per, R);
    ReqPlan* plan = (ReqPlan*)(p.ws + 256);
    if (tid == 0) taken_s = 0;
    // rows first: whether a request's rows end within n_rows depends on those before it
    int64_t rows = 0;
    for (int r = r0; r < r1; ++r) rows += max(p.new_len[r], 0);
    auto scan = [&](Sums v, Sums& total) {  // exclusive prefix over the block
        Sums in = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const Sums o = shfl_up(in, d);
            if (lane >= d) in = in + o;
        }
        __syncthreads();
        if (lane == 63) part[wv] = in;
        __syncthreads();
        Sums base = {0, 0, 0, 0};
        total = {0, 0, 0, 0};
        for (int k = 0; k < kPlanThreads / 64; ++k) {
            if (k == wv) base = total;
            total = total + part[k];
        }
        return Sums{base.rows + in.rows - v.rows, base.need + in.need - v.need, base.give + in.give - v.give,
                    base.pieces + in.pieces - v.pieces};
    };
    Sums all;
    const int64_t row0 = scan(Sums{rows, 0, 0, 0}, all).rows;
    auto one = [&](int r, int64_t& end, bool& fits, bool& rel) {
        const int64_t len = p.seq_len[r], n = p.new_len[r];
        end += max(n, (int64_t)0);
        fits = n >= 0 && len >= 0 && len + n <= ((int64_t)p.cols << p.bt_log) && end <= p.n_rows;
        rel = n < 0 && len >= 0;
        Sums s = {0, 0, 0, 0};
        const int held = held_pages(p, len);
        if (fits) s.need = max(held_pages(p, len + n) - held, 0);
        if (rel) s.give = held;
        return s;
    };
    Sums mine = {0, 0, 0, 0};
    int64_t end = row0;
    bool fits, rel;
    for (int r = r0; r < r1; ++r) mine = mine + one(r, end, fits, rel);
    Sums at = scan(mine, all);
    const int64_t given = all.give;
    const int64_t head = p.span[0], tail = p.span[1];
    // who is granted, and so the pieces
    int64_t take = at.need, taken = 0, pieces = 0;
    end = row0;
    auto grant = [&](int r, Sums& s) {
        s = one(r, end, fits, rel);
        const int64_t upto = take + s.need;
        const bool ok = fits && (s.need == 0 || upto <= tail - head);
        s.pieces = 0;
        if (ok && p.new_len[r] > 0) {
            const int64_t len = p.seq_len[r], n = p.new_len[r];
            s.pieces = ((len + n - 1) >> p.bt_log) - (len >> p.bt_log) + 1;
        }
        return ok;
    };
    for (int r = r0; r < r1; ++r) {
        Sums s;
        const bool ok = grant(r, s);
        take += s.need;
        if (ok && s.need > 0) taken = max(taken, take);
        pieces += s.pieces;
    }
    const int64_t piece0 = scan(Sums{0, 0, 0, pieces}, all).pieces;
    if (taken > 0) atomicMax((unsigned long long*)&taken_s, (unsigned long long)taken);
    take = at.need;
    int64_t give = at.give, piece = piece0;
    end = row0;
    for (int r = r0; r < r1; ++r) {
        Sums s;
        const int64_t begin = end;
        const bool ok = grant(r, s);
        plan[r] = {ok ? 1 : rel ? 2 : 0, (int32_t)piece, take, give};
        take += s.need;
        give += s.give;
        piece += s.pieces;
        p.cu[r] = (int32_t)min(begin, (int64_t)0x7fffffff);
        p.seq_out[r] = ok ? p.seq_len[r] + p.new_len[r] : rel ? 0 : p.seq_len[r];
        p.granted[r] = ok || rel;
        if (r == R - 1) p.cu[R] = (int32_t)min(end, (int64_t)0x7fffffff);
    }
    __syncthreads();
    if (tid == 0) {
        p.span_out[0] = head + taken_s;
        p.span_out[1] = min(tail + given, head + p.n_free);
        *(int64_t*)p.ws = all.pieces;
        if (R == 0) p.cu[0] = 0;
    }
}

__global__ __launch_bounds__(256) void rows_map_kernel(CacheRowsParams p, int row_blocks) {
    const ReqPlan* plan = (const ReqPlan*)(p.ws + 256);
    const int64_t head = p.span[0], tail = p.span[1];
    if ((int)blockIdx.x >= row_blocks) {  // pages given back: a wave a request
        const int r = ((int)blockIdx.x - row_blocks) * 4 + (threadIdx.x >> 6);
        if (r >= p.n_reqs || plan[r].state != 2) return;
        const int held = held_pages(p, p.seq_len[r]);
        const int64_t at = tail + plan[r].give;
        for (int j = threadIdx.x & 63; j < held; j += 64)
            if (at + j - head < p.n_free) p.ring[(uint64_t)(at + j) % (uint64_t)p.n_free] = p.table[r * p.table_st + j];
        return;
    }
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= p.n_rows) return;
    if (t < p.n_pieces && t >= *(const int64_t*)p.ws) {  // pieces past the last
        int4* z = (int4*)p.pieces + t;
        *z = make_int4(0, 0, 0, 0);
    }
    int lo = 0, hi = p.n_reqs;  // the first request whose rows end past t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int r = lo;
    int pos = -1;
    int64_t slot = -1;
    if (r < p.n_reqs && plan[r].state == 1) {
        const int bt = 1 << p.bt_log, row0 = p.cu[r], len = p.seq_len[r];
        pos = len + t - row0;
        const int b = pos >> p.bt_log, off = pos & (bt - 1), held = held_pages(p, len);
        int page;
        if (b < held) {
            page = p.table[r * p.table_st + b];
        } else {
            page = p.ring[(uint64_t)(head + plan[r].take + b - held) % (uint64_t)p.n_free];
            if (off == 0) p.table[r * p.table_st + b] = page;
        }
        slot = (int64_t)page * bt + off;
        if (t == row0 || off == 0) {
            const int k = plan[r].piece + b - (len >> p.bt_log);
            if (k < p.n_pieces) ((int4*)p.pieces)[k] = make_int4(t, min(bt - off, p.cu[r + 1] - t), page, off);
        }
    }
    p.req[t] = r < p.n_reqs ? r : -1;
    p.pos[t] = pos;
    p.slot[t] = slot;
}

// Up to kOneReqs requests in one launch: every block forms the sums for itself, in LDS, and writes its share of the rows.
constexpr int kOneReqs = 4096, kOnePer = kOneReqs / kPlanThreads;

struct OnePlan {
    int32_t cu[kOneReqs + 1];
    int32_t take[kOneReqs];   // its first page among those taken (granted) or given back (released)
    int32_t piece[kOneReqs];  // its first piece, -1: refused, -2: released
    unsigned long long part[kPlanThreads / 64];
    int taken, pieces;
};

// exclusive prefix over the block's first `waves` waves (others get nothing of use), and the total
__device__ __forceinline__ unsigned long long one_scan(OnePlan& sh, unsigned long long v, int waves, unsigned long long& total) {
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
    for (int k = 0; k < waves; ++k) {
        if (k == wv) base = total;
        total += sh.part[k];
    }
    return base + in - v;
}

__global__ __launch_bounds__(kPlanThreads) void rows_one_kernel(CacheRowsParams p) {
    __shared__ OnePlan sh;
    const int tid = threadIdx.x, R = p.n_reqs, bt = 1 << p.bt_log;
    const int per = ceil_div(R, kPlanThreads), waves = ceil_div(ceil_div(R, per), 64);
    const int64_t head = p.span[0], tail = p.span[1];
    const bool writer = blockIdx.x == 0;
    int64_t len[kOnePer], n[kOnePer];
    unsigned long long rows = 0, total;
    if (tid == 0) sh.taken = sh.pieces = 0;
#pragma unroll
    for (int i = 0; i < kOnePer; ++i) {
        const int r = tid * per + i;
        const bool in = i < per && r < R;
        len[i] = in ? p.seq_len[r] : -1;
        n[i] = in ? p.new_len[r] : 0;
        rows += max(n[i], (int64_t)0);
    }
    int64_t end = (int64_t)one_scan(sh, rows, waves, total);
    const int64_t row0 = end;
    // pages taken in the upper half, given back in the lower
    unsigned long long mine = 0;
    int need[kOnePer], held[kOnePer];
    bool fits[kOnePer];
#pragma unroll
    for (int i = 0; i < kOnePer; ++i) {
        end += max(n[i], (int64_t)0);
        held[i] = held_pages(p, len[i]);
        fits[i] = n[i] >= 0 && len[i] >= 0 && len[i] + n[i] <= ((int64_t)p.cols << p.bt_log) && end <= p.n_rows;
        need[i] = fits[i] ? max(held_pages(p, len[i] + n[i]) - held[i], 0) : 0;
        mine += ((unsigned long long)need[i] << 32) + (n[i] < 0 && len[i] >= 0 ? held[i] : 0);
    }
    unsigned long long at = one_scan(sh, mine, waves, total);
    const int64_t given = (int64_t)(uint32_t)total;
    int take = (int)(at >> 32), give = (int)(uint32_t)at, taken = 0;
    int pieces[kOnePer], all = 0;
    bool ok[kOnePer];
#pragma unroll
    for (int i = 0; i < kOnePer; ++i) {
        const int upto = take + need[i];
        ok[i] = fits[i] && (need[i] == 0 || upto <= tail - head);
        take = upto;
        if (ok[i] && need[i] > 0) taken = upto;
        pieces[i] = ok[i] && n[i] > 0 ? (int)(((len[i] + n[i] - 1) >> p.bt_log) - (len[i] >> p.bt_log)) + 1 : 0;
        all += pieces[i];
    }
    if (taken > 0) atomicMax(&sh.taken, taken);
    int piece = (int)one_scan(sh, (unsigned long long)all, waves, total);
    if (tid == 0) sh.pieces = (int)total;
    take = (int)(at >> 32);
    end = row0;
#pragma unroll
    for (int i = 0; i < kOnePer; ++i) {
        const int r = tid * per + i;
        if (i < per && r < R) {
            const bool rel = n[i] < 0 && len[i] >= 0;
            const int first = (int)min(end, (int64_t)0x7fffffff);
            sh.cu[r] = first;
            sh.take[r] = rel ? give : take;
            sh.piece[r] = ok[i] ? piece : rel ? -2 : -1;
            take += need[i];
            give += rel ? held[i] : 0;
            piece += pieces[i];
            end += max(n[i], (int64_t)0);
            const int last = (int)min(end, (int64_t)0x7fffffff);
            if (r == R - 1) sh.cu[R] = last;
            if (writer) {
                p.cu[r] = first;
                if (r == R - 1) p.cu[R] = last;
                p.seq_out[r] = (int32_t)(ok[i] ? len[i] + n[i] : rel ? 0 : len[i]);
                p.granted[r] = ok[i] || rel;
            }
        }
    }
    __syncthreads();
    if (writer && tid == 0) {
        p.span_out[0] = head + sh.taken;
        p.span_out[1] = min(tail + given, head + p.n_free);
    }
    // pages given back: a wave a request
    for (int r = blockIdx.x * (kPlanThreads / 64) + (tid >> 6); r < R; r += gridDim.x * (kPlanThreads / 64)) {
        if (sh.piece[r] != -2) continue;
        const int pages = held_pages(p, p.seq_len[r]);
        const int64_t to = tail + sh.take[r];
        for (int j = tid & 63; j < pages; j += 64)
            if (to + j - head < p.n_free) p.ring[(uint64_t)(to + j) % (uint64_t)p.n_free] = p.table[r * p.table_st + j];
    }
    const int t = blockIdx.x * kPlanThreads + tid;
    if (t >= p.n_rows) return;
    if (t < p.n_pieces && t >= sh.pieces) ((int4*)p.pieces)[t] = make_int4(0, 0, 0, 0);
    int lo = 0, hi = R;  // the first request whose rows end past t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sh.cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int r = lo;
    int pos = -1;
    int64_t slot = -1;
    if (r < R && sh.piece[r] >= 0) {
        const int first = sh.cu[r], old = p.seq_len[r];
        pos = old + t - first;
        const int b = pos >> p.bt_log, off = pos & (bt - 1), had = held_pages(p, old);
        int page;
        if (b < had) {
            page = p.table[r * p.table_st + b];
        } else {
            page = p.ring[(uint64_t)(head + sh.take[r] + b - had) % (uint64_t)p.n_free];
            if (off == 0) p.table[r * p.table_st + b] = page;
        }
        slot = (int64_t)page * bt + off;
        if (t == first || off == 0) {
            const int k = sh.piece[r] + b - (old >> p.bt_log);
            if (k < p.n_pieces) ((int4*)p.pieces)[k] = make_int4(t, min(bt - off, sh.cu[r + 1] - t), page, off);
        }
    }
    p.req[t] = r < R ? r : -1;
    p.pos[t] = pos;
    p.slot[t] = slot;
}

// --------------------------------------------------------------------- write
// A block takes one piece (rows of one request within one page), one head, keys or values: the largest
// finite magnitude of the rows gives the scale, codes held before the rows follow it where it grew, and
// the rows are rounded to e4m3.  A scale is a power of two, so that dividing by it is exact and codes
// that follow a larger one lose nothing above the subnormals.  Bound by memory: up to kKept vectors a thread
// stay in registers between the two passes, more are read again (16001 float32 rows of 8 heads of 64: 18 us, 4.6 TB/s;
// 21 with every row read twice).
constexpr int kKept = 4;

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void write_kernel(CacheWriteParams p) {
    constexpr int VEC = 16 / sizeof(T), WAVES = THREADS / 64;
    typedef T vec __attribute__((ext_vector_type(VEC), aligned(16)));
    __shared__ float red[WAVES], held_s;
    const int4 piece = ((const int4*)p.pieces)[blockIdx.x];
    const int row0 = piece.x, rows = piece.y, page = piece.z, off = piece.w;
    const int bt = 1 << p.c.bt_log, D = p.c.head_dim, g = blockIdx.y;
    // pieces past the last (no rows), and any that does not lie within the rows and one page
    if (rows <= 0 || row0 < 0 || rows > p.n_rows - row0 || page < 0 || page >= p.c.n_blocks || off < 0 || rows > bt - off) return;
    const int tid = threadIdx.x;
    const bool val = blockIdx.z != 0;
    const T* x = (const T*)(val ? p.v : p.k) + (int64_t)row0 * (val ? p.v_st : p.k_st) + (int64_t)g * (val ? p.v_sh : p.k_sh);
    const int64_t st = val ? p.v_st : p.k_st;
    const int64_t tile = (int64_t)page * p.c.n_kv + g;
    uint8_t* codes = (val ? p.c.v : p.c.k) + tile * bt * D;
    float* scale = (val ? p.c.vs : p.c.ks) + tile;
    float held = 0.f;  // (one thread reads the scale, and it alone writes it)
    if (tid == 0 && off > 0) held = *scale;
    const int per = D / VEC, shift = __builtin_ctz(per), n = rows * per;
    auto at = [&](int i) { return *(const vec*)(x + (i >> shift) * st + (i & (per - 1)) * VEC); };
    vec kept[kKept];
    float amax = 0.f;
    auto most = [&](const vec& v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float f = fabsf(to_float(v[e]));
            if (finite(f)) amax = fmaxf(amax, f);
        }
    };
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
        kept[k] = vec{};
        if (tid + k * THREADS < n) kept[k] = at(tid + k * THREADS);
    }
#pragma unroll
    for (int k = 0; k < kKept; ++k) most(kept[k]);
    for (int i = tid + kKept * THREADS; i < n; i += THREADS) most(at(i));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) amax = fmaxf(amax, wave_xor(amax, o));
    if constexpr (WAVES > 1) {
        if ((tid & 63) == 0) red[tid >> 6] = amax;
        if (tid == 0) held_s = held;
        __syncthreads();
        for (int k = 0; k < WAVES; ++k) amax = fmaxf(amax, red[k]);
        held = held_s;
    } else {
        held = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(held)));
    }
    const float s = fmaxf(scale_of(amax), held), inv = 1.f / s;
    if (s != held) {
        const float ratio = held * inv;
        uint32_t* u = (uint32_t*)codes;
        for (int i = tid; i < off * D / 4; i += THREADS) {
            float f[4];
            e4m3_x4(u[i], f);
            u[i] = to_e4m3_x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
        }
        if (tid == 0) *scale = s;
    }
    auto put = [&](int i, const vec& v) {
        typedef uint32_t words __attribute__((ext_vector_type(VEC / 4)));
        words o;
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
            o[e / 4] = to_e4m3_x4(to_float(v[e]) * inv, to_float(v[e + 1]) * inv, to_float(v[e + 2]) * inv,
                                  to_float(v[e + 3]) * inv);
        *(words*)(codes + off * D + i * VEC) = o;
    };
#pragma unroll
    for (int k = 0; k < kKept; ++k)
        if (tid + k * THREADS < n) put(tid + k * THREADS, kept[k]);
    for (int i = tid + kKept * THREADS; i < n; i += THREADS) put(i, at(i));
}

// ---------------------------------------------------------------------- read
// Row t of a packed batch is token start[r] + t - cu[r] of its request r.  A thread takes eight
// elements of one head, keys and values.
template <typename T>
__global__ __launch_bounds__(256) void read_kernel(CacheReadParams p) {
    typedef T vec __attribute__((ext_vector_type(8), aligned(16)));
    const int D = p.c.head_dim, per = p.c.n_kv * (D / 8);
    const int64_t n = (int64_t)p.n_rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int t = (int)(i / per), x = (int)(i - (int64_t)t * per), g = x / (D / 8), c = (x - g * (D / 8)) * 8;
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
                const int64_t tile = (int64_t)page * p.c.n_kv + g;
                const int64_t at = ((tile << p.c.bt_log) + (pos & ((1 << p.c.bt_log) - 1))) * D + c;
                const u32x2 ku = *(const u32x2*)(p.c.k + at), vu = *(const u32x2*)(p.c.v + at);
                const float ks = p.c.ks[tile], vs = p.c.vs[tile];
                float f[8];
                e4m3_x4(ku[0], f);
                e4m3_x4(ku[1], f + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = from_float<T>(f[e] * ks);
                e4m3_x4(vu[0], f);
                e4m3_x4(vu[1], f + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = from_float<T>(f[e] * vs);
            }
        }
        *(vec*)((T*)p.k + (int64_t)t * p.c.n_kv * D + g * D + c) = k;
        *(vec*)((T*)p.v + (int64_t)t * p.c.n_kv * D + g * D + c) = v;
    }
}

}  // namespace

// One launch while every block can form the sums for itself (and page counts fit 31 bits): 64 requests 7.7 us, 10.2 in two
// launches, 1500 requests with 32768 rows 11.8 and 16.4.  Past that one block forms the sums of all requests, whose time grows
// with them (a row each: 4096 requests in one launch 19 us, 4097 in two 27, 16384 126, 65536 528, 2^20 8.6 ms).
static bool rows_in_one(int n_reqs, int cols) { return n_reqs <= kOneReqs && (int64_t)n_reqs * cols < 0x7fffffff; }

size_t cache_rows_ws_bytes(int n_reqs, int cols) { return rows_in_one(n_reqs, cols) ? 0 : 256 + (size_t)n_reqs * sizeof(ReqPlan); }

hipError_t cache_rows_launch(const CacheRowsParams& p, hipStream_t stream) {
    if (rows_in_one(p.n_reqs, p.cols)) {
        const dim3 grid((unsigned)std::max(ceil_div(p.n_rows, kPlanThreads), 1));
        DSALT_LAUNCH("cache_rows", rows_one_kernel, grid, dim3(kPlanThreads), 0, stream, p);
        return hipGetLastError();
    }
    DSALT_LAUNCH("cache_rows_plan", rows_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
    const int row_blocks = ceil_div(p.n_rows, 256), blocks = row_blocks + ceil_div(p.n_reqs, 4);
    if (blocks > 0) DSALT_LAUNCH("cache_rows_map", rows_map_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, row_blocks);
    return hipGetLastError();
}

template <typename T>
static void write_pieces(const CacheWriteParams& p, hipStream_t stream) {
    // a wave where there are as many pieces as rows (200 rows, 16 heads of 128: 9.1 us with four waves, 6.8 with one), or a
    // whole page is what it keeps (16384 bfloat16 rows of 8 heads of 128 in pages of 16: 37 and 24)
    const int vecs = (p.c.head_dim * (int)sizeof(T) / 16) << p.c.bt_log;
    const bool wave = p.n_pieces == p.n_rows || vecs <= 64 * kKept;
    CacheWriteParams s = p;
    for (int64_t k = 0; k < p.n_pieces; k += s.n_pieces) {
        s.n_pieces = (int)std::min(p.n_pieces - k, kLaunchThreads / 256);
        s.pieces = p.pieces + 4 * k;
        const dim3 grid((unsigned)s.n_pieces, (unsigned)p.c.n_kv, 2);
        if (wave) DSALT_LAUNCH("cache_write", (write_kernel<T, 64>), grid, dim3(64), 0, stream, s);
        else DSALT_LAUNCH("cache_write", (write_kernel<T, 256>), grid, dim3(256), 0, stream, s);
    }
}

hipError_t cache_write_launch(const CacheWriteParams& p, hipStream_t stream) {
    if (p.n_pieces == 0 || p.n_rows == 0) return hipSuccess;
    switch (p.dtype) {
        case 0: write_pieces<float>(p, stream); break;
        case 1: write_pieces<bf16>(p, stream); break;
        default: write_pieces<f16>(p, stream); break;
    }
    return hipGetLastError();
}

hipError_t cache_read_launch(const CacheReadParams& p, hipStream_t stream) {
    if (p.n_rows == 0) return hipSuccess;
    const int64_t n = (int64_t)p.n_rows * p.c.n_kv * (p.c.head_dim / 8);
    const dim3 grid((unsigned)std::min((n + 255) / 256, (int64_t)1 << 20));
    switch (p.dtype) {
        case 0: DSALT_LAUNCH("cache_read", read_kernel<float>, grid, dim3(256), 0, stream, p); break;
        case 1: DSALT_LAUNCH("cache_read", read_kernel<bf16>, grid, dim3(256), 0, stream, p); break;
        default: DSALT_LAUNCH("cache_read", read_kernel<f16>, grid, dim3(256), 0, stream, p); break;
    }
    return hipGetLastError();
}

}  // namespace dsalt
