// Drawing one token per row of logits with temperature, top-k, top-p and min-p from given uniform numbers.
//   weights    e_i = exp((l_i - max l) / T), held as whole numbers w_i = round(2^40 e_i)
//   top-k      the k largest logits; equal logits in the order of their index
//   top-p      of those, the shortest run of largest ones whose weights reach p times their sum (at least one)
//   min-p      of those, the ones with e_i >= min_p (the largest always)
//   token      the first index, in index order, whose running sum of kept weights exceeds u times their total
// T <= 0: the largest logit's lowest index.  NaN and -inf are never drawn; a row of nothing else gives -1.
//
// Whole-number weights make every sum independent of its order (LDS atomics among them) and every comparison exact: the
// token is a function of the row, whichever threads it falls to.  exp is fp64 arithmetic (an fp32 one moves the border between
// two tokens by 1e-7, which over a flat row of 10^5 tokens changes one draw in a few hundred): 2^y by a polynomial that is
// 2^-45.9 off at most, below the weights' step.  2^-40 is below what a uniform fp32 number resolves.
//
// One workgroup per row, which reads the row again (out of the caches) for each of its passes; bound by the instructions per
// logit, not by HBM, so the passes are few and the exact work falls on few logits (256 rows of 128000 bf16: k = 50 30 us, top-p
// 61 us, no cut 50 us; the row's bytes alone 13 us; top-p of fp16 112 and of fp32 129 us, bytes 13 and 26):
//   top-k of few: the k-th largest of the lanes' own maxima is no larger than the k-th largest logit, so the logits from there on
//     (little more than k) hold all candidates: they are sorted in LDS and everything else -- top-p, min-p, the draw -- happens on
//     that list.
//   bf16 with another cut: the values are counted, and exponentials, sums and cuts are taken over the values that there are.
//   otherwise a cut (top-k, top-p) is found by a histogram over 2048 equal steps of (max - l) / T; the logits in the step where
//     the sum passes its goal are sorted (or, where they are more than the list holds, divided by eleven, eleven and ten bits of
//     their ordered bit pattern and then by index).  The draw sums pieces of 512 logits, then looks into one piece.
// Rows of at most 64 logits take a team of lanes each and rank by comparing all pairs.  For few long rows the maxima of groups of logits
// and the weights are taken by many workgroups first (split_rows, below).
#include "dnag_token_common.h"
#include <float.h>
#include <math.h>

#define SMP_BINS 2048
#define SMP_RANGE 29.0f          // 2^40 exp(-29) < 1/2: weights beyond (the last step) are 0
#define SMP_BITS 40
#define SMP_MAX_V (1 << 20)      // sums stay below 2^60
#define SMP_LIST 2048            // logits that are sorted in LDS
#define SMP_GROUP 128            // logits whose maximum is kept

typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    int64_t ld, rows;
    int V;
    const float *u;
    const float *temperature, *top_p, *min_p;          // per row or NULL
    const int32_t *top_k;
    double temperature1, top_p1, min_p1;               // where NULL
    int top_k1;
    int64_t *out;
    char *ws;                                          // few long rows: per row hist[SMP_BINS], a sum per piece, a maximum per group
    int64_t ws_row;
};
struct RowSet { double c, p, minw; int k; bool greedy; };      // c = log2(e) / T; minw = min_p 2^40
__device__ __forceinline__ RowSet row_set(const SampleArgs &a, int64_t row) {
    RowSet s;
    const double t = a.temperature ? (double)a.temperature[row] : a.temperature1;
    s.greedy = !(t > 0.0);
    s.c = fmin(1.4426950408889634074 / t, 1e300);      // finite: the largest logit's distance of 0 times it is 0
    s.p = a.top_p ? (double)a.top_p[row] : a.top_p1;
    const double q = a.min_p ? (double)a.min_p[row] : a.min_p1;
    s.minw = q == q ? q * 1099511627776.0 : 0.0;
    s.k = a.top_k ? a.top_k[row] : a.top_k1;
    return s;
}
// a logit as compared: NaN counts as -inf, -0 as +0
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ bool cuts_by_rank(const RowSet &s, int V) { return s.k > 0 && s.k < V; }
// The largest k that is sorted in a short list; beyond it the list's sorting costs more than cutting at a histogram.  Both in us, 64 rows
// of 100 logits, k = 20: 20 and 10; of 2000, 20: 10 and 10, 100: 17 and 10; of 8192, 100: 15 and 17, 200: 23 and 17; of 128000,
// 256: 35 and 50 (bf16), 400: 52 and 63 (fp32).
__host__ __device__ inline int short_list_k(int64_t V, bool counted) {
    const int most = counted ? 256 : 512, k = (int)(V / 256 < most ? V / 256 : most);
    return V <= 4096 ? (int)(V / 64) : k > 128 ? k : 128;
}
// order of the bit patterns = order of the values
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
// 2^40 exp((x - m) / T) before it is rounded, c = log2(e) / T; NaN and -inf give 2^-24 of a step.  Conversions and ldexp are slow
// beside additions in fp64, so the whole part of y is rounded off by adding 1.5 2^52 (it lands in the low bits) and added to
// the exponent as an integer.
__device__ __forceinline__ double raw_weight(float x, double m, double c) {
    const double y = fmax(((double)x - m) * c, -64.0);
    const double t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);               // f in [-1/2, 1/2]
    // 2^f: least relative error with p(0) = 1, fitted at 4000 points; 1.5e-14 off
    double p = 1.0148340400913933e-07;
    p = fma(p, f, 1.3258335536991744e-06);
    p = fma(p, f, 1.525299001687859e-05);
    p = fma(p, f, 0.00015403440883783207);
    p = fma(p, f, 0.0013333557625467886);
    p = fma(p, f, 0.009618129181164985);
    p = fma(p, f, 0.05550410866841576);
    p = fma(p, f, 0.24022650695722814);
    p = fma(p, f, 0.6931471805598851);
    p = fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + ((__double2loint(t) + SMP_BITS) << 20), __double2loint(p));
}
__device__ __forceinline__ u64 whole_weight(double v) {        // v in [0, 2^41): rounded by the addition's own rounding
    return (u64)__double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ float value_of_key(uint32_t k) { return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu)); }
// a row's weights and its steps of (max - l) / T; an infinite maximum leaves its equals alone: they weigh 1, everything else is
// below any cut
struct Weigh {
    float m;
    double md, c;
    bool inf;
    float per_step;
    __device__ __forceinline__ void set(float top, double scale) {
        m = top; c = scale; inf = m == INFINITY; md = inf ? 0.0 : (double)m;
        per_step = fminf((float)(c * 0.69314718055994531 * (double)(SMP_BINS / SMP_RANGE)), 1e30f);
    }
    __device__ __forceinline__ double raw(float x) const { return raw_weight(inf ? (x == m ? 0.f : -INFINITY) : x, md, c); }
    __device__ __forceinline__ u64 whole(float x) const { return whole_weight(raw(x)); }
    // never falls as x falls; the step is its whole part
    __device__ __forceinline__ float step(float x) const { return inf ? (x == m ? 0.f : SMP_BINS - 1.f) : fminf((m - x) * per_step, SMP_BINS - 1.f); }
    // min-p is a cut too: the smallest logit that weighs enough, by halving the ordered bit patterns up to the maximum's
    __device__ __forceinline__ float min_p_cut(double minw) const {
        uint32_t lo = 0x007fffffu, hi = ordered(m);    // lo: -inf, too light; hi: weighs enough, or is the largest anyway
        auto enough = [&](uint32_t key) { return raw(value_of_key(key)) >= minw; };
        const uint32_t near = ordered(clean((float)(md + (log2(minw) - SMP_BITS) / c)));       // almost always within two patterns
        if (near > lo + 2 && near + 2 < hi) {
            if (enough(near + 2)) hi = near + 2;
            if (!enough(near - 2)) lo = near - 2;
        }
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (enough(mid)) hi = mid;
            else lo = mid;
        }
        return value_of_key(hi);
    }
};
__device__ __forceinline__ u64 goal_of(double p, u64 total) {          // smallest whole number >= p total, 1 at least
    const double r = ceil(p * (double)total);
    return r >= 1.0 ? (r < (double)total ? (u64)r : total) : 1;
}
__device__ __forceinline__ u64 point_of(float u, u64 total) {          // the token is the first whose running sum exceeds this
    const double c = u >= 0.f ? (double)u * (double)total : 0.0;
    const u64 t = c < (double)total ? (u64)c : total - 1;
    return t < total ? t : total - 1;
}

// ---- rows of at most 64 logits: G lanes, one logit each ----------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(256) void sample_small_kernel(const SampleArgs a, int G) {
    const int lane = threadIdx.x & (G - 1);
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (row >= a.rows) return;
    const RowSet s = row_set(a, row);
    const float x = lane < a.V ? clean((float)((const T *)a.logits)[row * a.ld + lane]) : -INFINITY;
    float m = x;
    for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    int64_t token = -1;
    if (m > -INFINITY) {
        const bool live = x > -INFINITY;
        int rank = 0;
        for (int j = 0; j < G; ++j) {
            const float y = __shfl(x, (threadIdx.x & 63 & ~(G - 1)) + j, 64);
            rank += y > x || (y == x && j < lane);
        }
        int pick = rank == 0 ? lane : G;               // the largest logit's lowest index
        if (!s.greedy) {
            const double e = !live ? 0.0 : m == INFINITY ? (x == m ? 1099511627776.0 : 0.0) : raw_weight(x, (double)m, s.c);
            const u64 w = whole_weight(e);
            bool kept = live && (s.k <= 0 || rank < s.k);
            if (s.p < 1.0) {
                u64 total = 0, before = 0;
                const u64 mine = kept ? w : 0;
                for (int j = 0; j < G; ++j) {
                    const int from = (threadIdx.x & 63 & ~(G - 1)) + j;
                    const u64 wj = __shfl(mine, from, 64);
                    const int rj = __shfl(rank, from, 64);
                    total += wj;
                    before += rj < rank ? wj : 0;
                }
                kept = kept && before < goal_of(s.p, total);
            }
            kept = kept && (e >= s.minw || rank == 0);
            u64 sum = kept ? w : 0;
            for (int o = 1; o < G; o <<= 1) { const u64 b = __shfl_up(sum, o, 64); if (lane >= o) sum += b; }
            const u64 total = __shfl(sum, (threadIdx.x & 63) | (G - 1), 64);
            pick = sum > point_of(a.u[row], total) ? lane : G;
        }
        for (int o = G / 2; o > 0; o >>= 1) { const int b = __shfl_xor(pick, o, 64); pick = b < pick ? b : pick; }
        token = pick;
    }
    if (lane == 0) a.out[row] = token;
}

// ---- few long rows: what the row's workgroup would read them for, by many ------------------------------------------------
__host__ __device__ inline int64_t ws_pieces(int64_t V) { return (V + 511) / 512; }
__host__ __device__ inline int64_t ws_groups(int64_t V) { return (V + SMP_GROUP - 1) / SMP_GROUP; }
struct RowSpace {
    u64 *hist, *piece;
    float *top;                                        // the largest logit of every SMP_GROUP
    __device__ __forceinline__ RowSpace(const SampleArgs &a, int64_t row) {
        hist = (u64 *)(a.ws + row * a.ws_row);
        piece = hist + SMP_BINS;
        top = (float *)(piece + ws_pieces(a.V));
    }
};
// eight logits from c on as they are; past the end the row's last eight, with what lies before c set to -inf
template <class T> __device__ __forceinline__ f8 last8(typename Vec8<T>::type raw, int c, int V) {
    f8 v = widen<T>(raw);
    if (c + 8 > V) {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e < 8 - (V - c)) v[e] = -INFINITY;
    }
    return v;
}
template <class T>
__global__ __launch_bounds__(256) void sample_groups_kernel(const SampleArgs a) {
    const RowSpace w(a, blockIdx.y);
    const T *l = (const T *)a.logits + blockIdx.y * a.ld;
    const int i = blockIdx.x * 256 + threadIdx.x, c = i * 8;
    for (int b = i; b < SMP_BINS; b += gridDim.x * 256) w.hist[b] = 0;
    const f8 v = last8<T>(load8_raw(l + (c + 8 <= a.V ? c : a.V - 8)), c, a.V);
    float m = fmaxf(-INFINITY, max8(v));
    m = team_max<SMP_GROUP / 8>(m);
    if (c < a.V && (threadIdx.x & (SMP_GROUP / 8 - 1)) == 0) w.top[c / SMP_GROUP] = clean(m);
}
// Without a cut by rank: with top-p the histogram, otherwise every piece's kept weight.  The sums are whole numbers, so neither depends on order.
template <class T>
__global__ __launch_bounds__(256) void sample_weights_kernel(const SampleArgs a) {
    constexpr int EACH = 2;                            // pieces of a wave
    typedef typename Vec8<T>::type raw8;
    __shared__ u64 hist[SMP_BINS];
    __shared__ float wf[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.V;
    const RowSet s = row_set(a, blockIdx.y);
    if (s.greedy || cuts_by_rank(s, V)) return;
    const RowSpace w(a, blockIdx.y);
    const T *l = (const T *)a.logits + blockIdx.y * a.ld;
    const int p0 = (blockIdx.x * 4 + wave) * EACH;
    raw8 raw[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int c = (p0 + j) * 512 + lane * 8;
        raw[j] = load8_raw(l + (c + 8 <= V ? c : V - 8));
    }
    const bool nucleus = !__is_same(T, tbf16) && s.p < 1.0;    // bf16 rows are not split where top-p is asked for
    if (nucleus) for (int b = tid; b < SMP_BINS; b += 256) hist[b] = 0;
    float m = -INFINITY;
    const int groups = (int)ws_groups(V);
    for (int g = tid; g < groups; g += 256) m = fmaxf(m, w.top[g]);
    m = team_max<64>(m);
    if (lane == 0) wf[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(wf[0], wf[1]), fmaxf(wf[2], wf[3]));
    if (m == -INFINITY) return;
    Weigh weigh;
    weigh.set(m, s.c);
    if (nucleus) {
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const f8 v = last8<T>(raw[j], (p0 + j) * 512 + lane * 8, V);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = weigh.step(v[e]);
                if (q < SMP_BINS - 1.f) atomicAdd(&hist[(int)q], weigh.whole(v[e]));
            }
        }
        __syncthreads();
        for (int b = tid; b < SMP_BINS; b += 256) if (hist[b]) atomicAdd(&w.hist[b], hist[b]);
        return;
    }
    const float from = s.minw > 0.0 ? weigh.min_p_cut(s.minw) : -INFINITY;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const f8 v = last8<T>(raw[j], (p0 + j) * 512 + lane * 8, V);
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += weigh.whole(v[e] >= from ? v[e] : -INFINITY);
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0 && (p0 + j) * 512 < V) w.piece[p0 + j] = sum;
    }
}

// ---- one workgroup per row -----------------------------------------------------------------------------------------------
struct Cut { float x; int at; };   // kept: larger logits, and equal ones up to index `at`

// SPLIT: sample_groups_kernel and, where it applies, sample_weights_kernel have run
template <class T, int NTHR, bool SPLIT>
__global__ __launch_bounds__(NTHR) void sample_row_kernel(const SampleArgs a) {
    constexpr int NW = NTHR / 64, PER = SMP_BINS / NTHR;
    constexpr bool COUNTED = __is_same(T, tbf16);
    extern __shared__ u64 piece[];                     // sums of 512 logits each, for the draw
    __shared__ u64 hist[SMP_BINS];                     // histogram, or the list of logits that is sorted
    static_assert(SMP_LIST <= SMP_BINS, "the list shares the histogram's memory");
    __shared__ float queue[NW][512];
    __shared__ u64 ws[NW];
    __shared__ float wf[NW];
    __shared__ int wi[2][8 * NW];
    __shared__ u64 found[3];                           // bin, sum before it, sum in it
    __shared__ int at_found, listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const T *l = (const T *)a.logits + row * a.ld;
    const int V = a.V;
    const RowSet s = row_set(a, row);
    // f(first index, eight logits as they are), called by whole waves: a lane past the end has -inf, and the row's last piece
    // that is shorter than eight comes as the row's last eight with what was seen before set to -inf.  A rolled loop with three
    // pieces under way ahead of the one that is worked on: a workgroup runs through each pass once, so what counts is the code's size (with
    // the pieces unrolled the passes waited for instructions).
    auto each8 = [&](auto f) {
        typedef typename Vec8<T>::type raw8;
        constexpr int STEP = NTHR * 8;
        auto ask = [&](int c) { return load8_raw(l + (c + 8 <= V ? c : V - 8)); };
        int c = tid * 8;
        raw8 r0 = ask(c), r1 = ask(c + STEP), r2 = ask(c + 2 * STEP);
#pragma unroll 1
        for (; __builtin_amdgcn_readfirstlane(c) < V; c += STEP) {
            const raw8 now = r0;
            r0 = r1;
            r1 = r2;
            r2 = ask(c + 3 * STEP);
            f(c + 8 <= V ? c : V - 8, last8<T>(now, c, V));
        }
    };
    const RowSpace ws_row(a, row);
    const int groups = (int)ws_groups(V);
    float m = -INFINITY;                               // the row's largest logit
    Weigh weigh;
    auto weight_raw = [&](float x) { return weigh.raw(x); };
    auto weight = [&](float x) { return weigh.whole(x); };
    auto wave_scan = [&](u64 v) {                      // inclusive
        for (int o = 1; o < 64; o <<= 1) { const u64 b = __shfl_up(v, o, 64); if (lane >= o) v += b; }
        return v;
    };
    auto block_before = [&](u64 sum, u64 &total) {     // sum over the lanes before this one
        const u64 inc = wave_scan(sum);
        __syncthreads();
        if (lane == 63) ws[wave] = inc;
        __syncthreads();
        u64 before = inc - sum;
        total = 0;
        for (int w = 0; w < NW; ++w) { if (w < wave) before += ws[w]; total += ws[w]; }
        return before;
    };
    // The list: (ordered bits, ~index) in hist[0 .. n), sorted to falling logits and rising indices.
    auto entry = [&](float x, int i) { return (u64)ordered(x) << 32 | (uint32_t)~i; };
    auto value_of = [&](u64 e) { return value_of_key((uint32_t)(e >> 32)); };
    auto index_of = [&](u64 e) { return (int)~(uint32_t)e; };
    auto sort_falling = [&](int n) {
        __syncthreads();
        if (n <= (NTHR < 512 ? NTHR : 512)) {          // by counting what is larger (no barriers between steps), `parts` lanes for each
            int shift = 0;
            while (shift < 6 && (n << (shift + 1)) <= NTHR) ++shift;
            if (shift < 2) shift = 0;
            const int i = tid >> shift, parts = 1 << shift;
            const u64 x = i < n ? hist[i] : 0;
            int r = 0;
            if (shift == 0) {
                if (i < n)
#pragma unroll 8
                    for (int j = 0; j < n; ++j) { const u64 y = hist[j]; r += y > x || (y == x && j < i); }
            } else if (i < n)
                for (int j = tid & (parts - 1); j < n; j += parts) { const u64 y = hist[j]; r += y > x || (y == x && j < i); }
            for (int o = 1; o < parts; o <<= 1) r += __shfl_xor(r, o, 64);
            __syncthreads();
            if (i < n && !(tid & (parts - 1))) hist[r] = x;
            __syncthreads();
            return;
        }
        int n2 = 2;
        while (n2 < n) n2 *= 2;
        for (int i = n + tid; i < n2; i += NTHR) hist[i] = 0;
        for (int k = 2; k <= n2; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                __syncthreads();
                for (int p = tid; p < n2 / 2; p += NTHR) {
                    const int i = 2 * p - (p & (j - 1));
                    const u64 x = hist[i], y = hist[i + j];
                    if ((x < y) == ((i & k) == 0)) { hist[i] = y; hist[i + j] = x; }
                }
            }
        __syncthreads();
    };
    auto collect = [&](float from, float to, auto take) {  // logits in [from, to] that `take` wants, in any order; their number (the list may hold fewer)
        from = fmaxf(from, -FLT_MAX);                  // never -inf: neither drawn nor there (each8)
        __syncthreads();
        if (tid == 0) { listed = 0; at_found = 0; }
        __syncthreads();
        auto look = [&](int c, const f8 &v) {
            if (!(max8(v) >= from)) return;
            uint32_t hit = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) hit |= (v[e] >= from && v[e] <= to ? 1u : 0u) << e;
            for (; hit; hit &= hit - 1) {              // few
                const int b = __ffs(hit) - 1, i = c + b;
                float x = v[0];                        // chosen among the registers: the wave would wait for a load
#pragma unroll
                for (int e = 1; e < 8; ++e) x = e == b ? v[e] : x;
                x = clean(x);
                if (!take(x, i)) continue;
                const int at = atomicAdd(&listed, 1);
                if (at < SMP_LIST) hist[at] = entry(x, i);
            }
        };
        if constexpr (SPLIT) {                         // only the groups that reach so far
            int *group = (int *)&queue[0][0];
            static_assert(SMP_MAX_V / SMP_GROUP <= NW * 512, "the groups share the queue's memory");
            for (int g = tid; g < groups; g += NTHR)
                if (ws_row.top[g] >= from) group[atomicAdd(&at_found, 1)] = g;
            __syncthreads();
            const int n = at_found;
            constexpr int TEAM = SMP_GROUP / 8;
            for (int q = tid / TEAM; q < n; q += NTHR / TEAM) {
                const int c = group[q] * SMP_GROUP + (tid & (TEAM - 1)) * 8;
                if (c < V) look(c + 8 <= V ? c : V - 8, last8<T>(load8_raw(l + (c + 8 <= V ? c : V - 8)), c, V));
            }
        } else each8(look);
        __syncthreads();
        return listed;
    };
    Cut cut{-INFINITY, -1};                            // everything that can be drawn
    const bool short_list = s.k > 0 && s.k < V && s.k <= short_list_k(V, COUNTED);
    bool done = false;                                 // `cut` is final and `piece` holds the kept weights' sums
    const int pieces = (V + 511) / 512;
    auto inside = [&](const Cut &c, float x, int i) { return x > c.x || (x == c.x && i <= c.at); };
    // ---- bf16: few values, counted ---------------------------------------------------------------------------------------
    // A row of bf16 logits holds few different values.  Those of magnitude 2^-9 .. 2^9 are counted (4608 slots in falling order), the
    // exponentials, sums and cuts are taken over the slots, and the draw looks its weights up.  What is nearer to 0 (slot HALF)
    // is listed and weighed one by one.  Rows that do not fit -- a logit from 512 on, a list that is too short, a cut between the
    // listed ones -- go the general way.  256 rows of 128000, top-p with min-p: 120 us the general way, 69 this way.
    const bool ranks = cuts_by_rank(s, V);
    if constexpr (NTHR == 1024 && COUNTED && !SPLIT) {
        constexpr int HALF = 18 * 128, EACH = 5, SLOTS = EACH * NTHR;
        static_assert(2 * HALF + 1 <= SLOTS && sizeof(uint32_t) * SLOTS <= sizeof(queue), "slots");
        uint32_t *count = (uint32_t *)&queue[0][0];
        u64 *table = piece + pieces;
        float *near = (float *)hist;                   // [SMP_LIST], then [SMP_LIST] indices of equal logits at the cut
        int *ties = (int *)(near + SMP_LIST);
        auto slot_of = [&](float x) {
            const uint32_t h = __float_as_uint(x) >> 16, i = (h & 0x7fffu) - 0x3b00u;
            return i < (uint32_t)HALF ? (int)(h & 0x8000u ? HALF + 1 + i : HALF - 1 - i) : -1;
        };
        auto value_at = [&](int r) { return __uint_as_float((r < HALF ? 0x3b00u + (HALF - 1 - r) : 0xbb00u + (r - HALF - 1)) << 16); };
        if (!s.greedy && (ranks || s.p < 1.0) && !short_list) {
            for (int r = tid; r < SLOTS; r += NTHR) count[r] = 0;
            if (tid == 0) { listed = 0; at_found = 0; found[0] = SLOTS; found[1] = SLOTS; found[2] = 0; }
            __syncthreads();
            int odd = 0;                               // 1: a logit below -512, 2: one from 512 on
            each8([&](int, const f8 &v) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = slot_of(v[e]);
                    if (r >= 0) atomicAdd(&count[r], 1u);
                    else if (fabsf(v[e]) < 1.0f) {
                        const int at = atomicAdd(&listed, 1);
                        if (at < SMP_LIST) near[at] = clean(v[e]);
                    } else if (v[e] > -INFINITY) odd |= v[e] > 0.f ? 2 : 1;
                }
            });
            if (odd) atomicOr(&at_found, odd);
            __syncthreads();
            const int n_near = listed;
            bool fits = n_near <= SMP_LIST && !(at_found & 2);
            // the maximum: the first slot that is not empty, or among the listed ones
            uint32_t cnt[EACH];
            int first = SLOTS;
#pragma unroll
            for (int q = EACH - 1; q >= 0; --q) {
                const int r = tid * EACH + q;
                cnt[q] = r == HALF ? (uint32_t)n_near : count[r];
                if (cnt[q] && r != HALF) first = r;
            }
            float top = first < SLOTS ? value_at(first) : -INFINITY;
            if (fits) for (int i = tid; i < n_near; i += NTHR) top = fmaxf(top, near[i]);
            top = team_max<64>(top);
            if (lane == 0) wf[wave] = top;
            __syncthreads();
            for (int w = 0; w < NW; ++w) top = fmaxf(top, wf[w]);
            // logits below -512 may be left out where they weigh nothing
            fits = fits && top > -INFINITY && (!(at_found & 1) || ((double)top + 512.0) * s.c > 42.0) && !(s.minw > 1099511627776.0);
            if (fits) {
                m = top;
                weigh.set(m, s.c);
                u64 w[EACH], sum = 0, total, near_sum;
                bool light[EACH];                      // min-p drops the slot
                u64 near_mine = 0;
                int heavy = 0;
                for (int i = tid; i < n_near; i += NTHR) { const double v = weight_raw(near[i]); near_mine += whole_weight(v); heavy += v >= s.minw; }
                block_before(near_mine, near_sum);
                u64 heavies;
                block_before(heavy, heavies);
#pragma unroll
                for (int q = 0; q < EACH; ++q) {
                    const int r = tid * EACH + q;
                    const double v = cnt[q] && r != HALF ? weight_raw(value_at(r)) : 0.0;
                    w[q] = whole_weight(v);
                    light[q] = cnt[q] && (r == HALF ? heavies == 0 : !(v >= s.minw));
                    table[r] = w[q];
                }
                bool mixed = n_near > 0 && heavies > 0 && heavies < (u64)n_near;      // a cut between the listed ones
                int c_slot = SLOTS, c_ties = 0;        // kept: slots before c_slot, and c_ties logits of it
                if (ranks) {
                    u64 n = 0, all;
#pragma unroll
                    for (int q = 0; q < EACH; ++q) n += cnt[q];
                    u64 before = block_before(n, all);
#pragma unroll
                    for (int q = 0; q < EACH; ++q) {
                        if (before < (u64)s.k && before + cnt[q] >= (u64)s.k) { found[0] = tid * EACH + q; found[2] = s.k - before; }
                        before += cnt[q];
                    }
                    __syncthreads();
                    c_slot = (int)found[0];
                    c_ties = c_slot < SLOTS ? (int)found[2] : 0;
                    mixed = mixed || (c_slot == HALF && c_ties < n_near);
                    __syncthreads();
                }
                if (s.p < 1.0) {
                    u64 part[EACH];
#pragma unroll
                    for (int q = 0; q < EACH; ++q) {
                        const int r = tid * EACH + q;
                        const u64 n = r < c_slot ? cnt[q] : r == c_slot ? (u64)c_ties : 0;
                        part[q] = r == HALF ? (n ? near_sum : 0) : n * w[q];
                        sum += part[q];
                    }
                    u64 before = block_before(sum, total);
                    const u64 goal = goal_of(s.p, total);
#pragma unroll
                    for (int q = 0; q < EACH; ++q) {
                        if (before < goal && before + part[q] >= goal) {
                            const int r = tid * EACH + q;
                            found[1] = r;
                            found[2] = r == HALF ? (before + part[q] == goal ? (u64)n_near : 0) : (goal - before + w[q] - 1) / w[q];
                        }
                        before += part[q];
                    }
                    __syncthreads();
                    c_slot = (int)found[1];            // top-p keeps a part of what top-k kept: its cut is the earlier one
                    c_ties = (int)found[2];
                    mixed = mixed || (c_slot == HALF && c_ties == 0);
                    __syncthreads();
                }
                if (s.minw > 0.0) {
                    if (tid == 0) found[0] = SLOTS;
                    __syncthreads();
                    int lightest = SLOTS;
#pragma unroll
                    for (int q = EACH - 1; q >= 0; --q) if (light[q]) lightest = tid * EACH + q;
                    for (int o = 32; o > 0; o >>= 1) { const int b = __shfl_xor(lightest, o, 64); lightest = b < lightest ? b : lightest; }
                    if (lane == 0) atomicMin(&found[0], (u64)lightest);
                    __syncthreads();
                    if ((int)found[0] <= c_slot) { c_slot = (int)found[0]; c_ties = 0; }
                    __syncthreads();
                }
                if (!mixed) {
                    // equal logits at the cut of which only some are kept are listed by the draw's pass
                    const bool near_kept = HALF < c_slot || (HALF == c_slot && c_ties > 0);
                    const int c_count = c_slot < SLOTS && c_slot != HALF ? (int)count[c_slot] : 0;
                    const bool some = c_slot < SLOTS && c_slot != HALF && c_ties > 0 && c_ties < c_count;
                    const u64 c_weight = c_slot < SLOTS ? table[c_slot] : 0;
                    __syncthreads();
                    for (int r = c_slot + (c_ties > 0 && !some ? 1 : 0) + tid; r < SLOTS; r += NTHR) table[r] = 0;
                    for (int q = tid; q < pieces; q += NTHR) piece[q] = 0;
                    if (tid == 0) { listed = 0; at_found = -1; }
                    __syncthreads();
                    each8([&](int i0, const f8 &v) {
                        u64 sum = 0;
                        uint32_t hit = 0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int r = slot_of(v[e]);
                            if (r >= 0) sum += table[r];
                            else if (near_kept && fabsf(v[e]) < 1.0f) sum += weight(v[e]);
                            hit |= (r == c_slot ? 1u : 0u) << e;
                        }
                        if (some)
                            for (; hit; hit &= hit - 1) {
                                const int at = atomicAdd(&listed, 1);
                                if (at < SMP_LIST) ties[at] = i0 + __ffs(hit) - 1;
                            }
                        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
                        if (lane == 0) piece[(i0 + 7) >> 9] = sum;
                    });
                    __syncthreads();
                    const int n = listed;
                    if (n <= SMP_LIST) {
                        for (int i = tid; i < n; i += NTHR) {          // those of the lowest indices
                            const int mine_at = ties[i];
                            int rank = 0;
#pragma unroll 8
                            for (int j = 0; j < n; ++j) rank += ties[j] < mine_at;
                            if (rank < c_ties) atomicAdd(&piece[mine_at >> 9], c_weight);
                            if (rank == c_ties - 1) at_found = mine_at;
                        }
                        __syncthreads();
                        if (c_slot == HALF) cut = near_kept ? Cut{-0.001953125f, -1} : Cut{0.001953125f, 0x7fffffff};
                        else if (c_slot < SLOTS) cut = Cut{value_at(c_slot), some ? at_found : c_ties > 0 ? 0x7fffffff : -1};
                        done = true;
                    }
                }
            }
            __syncthreads();
        }
    }
    float mine = -INFINITY;                            // this lane's largest logit (the maximum passes NaN over)
    if (!done) {
        if constexpr (SPLIT) {
            for (int g = tid; g < groups; g += NTHR) mine = fmaxf(mine, ws_row.top[g]);
        } else {
            each8([&](int, const f8 &v) { mine = fmaxf(mine, max8(v)); });
            mine = clean(mine);
        }
        m = team_max<64>(mine);
        __syncthreads();
        if (lane == 0) wf[wave] = m;
        if (tid == 0) { at_found = 0x7fffffff; listed = 0; }
        __syncthreads();
        for (int w = 0; w < NW; ++w) m = fmaxf(m, wf[w]);
        if (m == -INFINITY) { if (tid == 0) a.out[row] = -1; return; }
        if (s.greedy) {
            if constexpr (SPLIT) {
                for (int g = tid; g < groups; g += NTHR) if (ws_row.top[g] == m) { atomicMin(&at_found, g); break; }
                __syncthreads();
                if (wave == 0) {
                    const int c = at_found * SMP_GROUP + lane * 2;
                    const uint64_t even = __ballot(c < V && (float)l[c < V ? c : V - 1] == m), odd = __ballot(c + 1 < V && (float)l[c + 1 < V ? c + 1 : V - 1] == m);
                    const int i0 = even ? 2 * (__ffsll((long long)even) - 1) : SMP_GROUP, i1 = odd ? 2 * __ffsll((long long)odd) - 1 : SMP_GROUP;
                    if (lane == 0) a.out[row] = at_found * SMP_GROUP + (i0 < i1 ? i0 : i1);
                }
                return;
            }
            if (mine == m) {
                int first = 0x7fffffff;
                each8([&](int c, const f8 &v) {
#pragma unroll
                    for (int e = 7; e >= 0; --e) if (v[e] == m && c + e < first) first = c + e;
                });
                atomicMin(&at_found, first);
            }
            __syncthreads();
            if (tid == 0) a.out[row] = at_found;
            return;
        }
        weigh.set(m, s.c);
    }
    // ---- top-k on a short list ---------------------------------------------------------------------------------------
    if (!done && short_list) {
        // A bound that k of the lanes' maxima reach, and not many more: the ordered bits of the maximum less a power of two (2^23 is an
        // octave), eight powers at a time; then, while that leaves too many, the ninth of the range that holds the k-th largest
        // (bounds that left up to 2 k + 256 made the list's sorting the longest step: 32 rows of 16384, k = 50, 25 us; now 13).
        const uint32_t key = ordered(mine), top_key = ordered(m);
        uint32_t low = 0, high = top_key;              // at least k reach low, fewer than k reach high (but where low is high)
        int reach = 0, turn = 0;
        auto eight = [&](auto bound) {                 // the first of bound(0 .. 7) that k reach, 8 if none; their number in `reach`
            int *buf = wi[turn++ & 1];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int c = __popcll(__ballot(key >= bound(q)));
                if (lane == 0) buf[q * NW + wave] = c;
            }
            __syncthreads();
            for (int q = 0; q < 8; ++q) {
                int n = 0;
#pragma unroll
                for (int w = 0; w < NW; ++w) n += buf[q * NW + w];
                if (n >= s.k) { reach = n; return q; }
            }
            return 8;
        };
        for (int b = 18; b < 32 && reach == 0; b += 8) {
            auto below = [&](int q) { return b + q >= 0 && b + q < 32 && top_key > 1u << (b + q) ? top_key - (1u << (b + q)) : 0u; };
            const int q = eight(below);
            if (q > 0) high = below(q - 1);
            if (q < 8) low = below(q);
        }
        while (reach > s.k + s.k / 4 + 16 && high - low > 1) {
            const uint32_t step = (high - low) / 9 > 0 ? (high - low) / 9 : 1, was = low, up = high;
            auto even = [&](int q) { const uint32_t x = was + (8 - q) * step; return x < up ? x : up; };
            const int q = eight(even);
            if (q > 0) high = even(q - 1);
            if (q < 8) low = even(q);
        }
        // as a logit (what lies between -0 and +0 becomes 0, a key below every logit's becomes -inf)
        float from = low <= 0x007fffffu ? -INFINITY : value_of((u64)low << 32);
        if (from == 0.f) from = 0.f;
        const int n = collect(from, INFINITY, [](float, int) { return true; });
        if (n <= SMP_LIST) {
            sort_falling(n);
            const int k = n < s.k ? n : s.k;
            constexpr int EACH = SMP_LIST / NTHR;      // consecutive entries of a lane
            u64 w[EACH], e[EACH], sum = 0, total;
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                const int i = tid * EACH + q;
                e[q] = i < k ? hist[i] : 0;
                const double v = i < k ? weight_raw(value_of(e[q])) : 0.0;
                w[q] = whole_weight(v);
                sum += w[q];
                if (!(v >= s.minw) && i != 0) e[q] = 0;          // fails min-p; its weight still counts for top-p
            }
            const u64 before = block_before(sum, total);
            const u64 goal = s.p < 1.0 ? goal_of(s.p, total) : ~0ull;
            __syncthreads();
            u64 run = before;
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                const int i = tid * EACH + q;
                if (i < k) hist[i] = e[q] != 0 && run < goal ? ((u64)(uint32_t)e[q] << 32 | (e[q] >> 32)) : 0;      // ~index first: rising indices
                run += w[q];
            }
            sort_falling(k);                           // by index; what is not kept goes to the end
            sum = 0;
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                const int i = tid * EACH + q;
                e[q] = i < k ? hist[i] : 0;
                w[q] = e[q] ? weight(value_of(e[q] << 32)) : 0;
                sum += w[q];
            }
            run = block_before(sum, total);
            const u64 t = point_of(a.u[row], total);
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                if (run <= t && run + w[q] > t) a.out[row] = index_of(e[q] >> 32);
                run += w[q];
            }
            return;
        }
    }
    // ---- any cut -----------------------------------------------------------------------------------------------------
    const float per_step = weigh.per_step;
    auto step_of = [&](float x) { return weigh.step(x); };
    auto clear = [&]() {
        __syncthreads();
        for (int b = tid; b < SMP_BINS; b += NTHR) hist[b] = 0;
        __syncthreads();
    };
    // the first bin whose running sum reaches the goal; goal(total) is asked once the total is known
    auto scan = [&](auto goal) {
        __syncthreads();
        u64 h[PER], sum = 0, total;
#pragma unroll
        for (int q = 0; q < PER; ++q) { h[q] = hist[tid * PER + q]; sum += h[q]; }
        if (tid == 0) found[0] = SMP_BINS;
        u64 before = block_before(sum, total);
        const u64 want = goal(total);
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            if (before < want && before + h[q] >= want) { found[0] = tid * PER + q; found[1] = before; found[2] = h[q]; }
            before += h[q];
        }
        __syncthreads();
        return want;
    };
    // cut where the sum of wt over the elements that `was` keeps reaches its goal
    auto find_cut = [&](const Cut &was, bool counts, auto wt, auto goal) {
        const bool any = was.x == -INFINITY;
        if (SPLIT && !ranks) {                         // sample_weights_kernel has made it
            __syncthreads();
            for (int b = tid; b < SMP_BINS; b += NTHR) hist[b] = ws_row.hist[b];
        } else {
        clear();
        each8([&](int i0, const f8 &v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = step_of(v[e]);
                const u64 w = wt(v[e]);
                if ((counts ? v[e] > -INFINITY : q < SMP_BINS - 1.f) && (any || inside(was, v[e], i0 + e))) atomicAdd(&hist[(int)q], w);
            }
        });
        }
        u64 want = scan(goal);
        if (found[0] == SMP_BINS) return was;          // the goal is not reached: all are kept
        const int step = (int)found[0];
        want -= found[1];
        // bounds of the step, a little wide, spare most logits the exact test
        const float wide = (float)step / per_step, far = (float)(step + 1) / per_step, slack = (fabsf(m) + far) * 1e-6f;
        const float to = m - wide + slack, from = step == SMP_BINS - 1 ? -INFINITY : m - far - slack;
        const int n = collect(from == from ? from : -INFINITY, to == to ? to : INFINITY, [&](float x, int i) { return inside(was, x, i) && (int)step_of(x) == step; });
        if (n <= SMP_LIST) {                           // the first of the sorted ones whose running sum reaches what is left
            sort_falling(n);
            constexpr int EACH = SMP_LIST / NTHR;
            u64 w[EACH], sum = 0, total;
#pragma unroll
            for (int q = 0; q < EACH; ++q) { const int i = tid * EACH + q; w[q] = i < n ? wt(value_of(hist[i])) : 0; sum += w[q]; }
            u64 run = block_before(sum, total);
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                if (run < want && run + w[q] >= want) found[0] = hist[tid * EACH + q];
                run += w[q];
            }
            __syncthreads();
            const u64 e = found[0];
            __syncthreads();
            return Cut{value_of(e), index_of(e)};
        }
        uint32_t prefix = 0;
        for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
            const int bits = shift == 0 ? 10 : 11;
            clear();
            each8([&](int i0, const f8 &v) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (inside(was, v[e], i0 + e) && (int)step_of(v[e]) == step) {
                        const uint32_t k = ordered(clean(v[e]));
                        if (shift == 21 || (k >> (shift + bits)) == prefix)
                            atomicAdd(&hist[(1 << bits) - 1 - ((k >> shift) & ((1u << bits) - 1))], wt(v[e]));
                    }
            });
            scan([&](u64) { return want; });
            prefix = (prefix << bits) | ((1u << bits) - 1 - (uint32_t)found[0]);
            want -= found[1];
        }
        // equal logits: as many as it takes, by index
        const float x = value_of((u64)prefix << 32);
        const u64 w1 = wt(x);
        u64 need = (want + w1 - 1) / w1;               // the need-th of them is the last one kept
        for (int c0 = 0; c0 < V; c0 += NTHR * 8) {
            const int i0 = c0 + tid * 8;
            uint32_t hit = 0;
            if (i0 < V) {
                const f8 v = load8_n(l + i0, V - i0, -INFINITY);
#pragma unroll
                for (int e = 0; e < 8; ++e) if (v[e] == x && inside(was, v[e], i0 + e)) hit |= 1u << e;
            }
            u64 all;
            const u64 n1 = __popc(hit), before = block_before(n1, all);
            if (before < need && before + n1 >= need) {
                for (u64 q = before + 1; q < need; ++q) hit &= hit - 1;
                at_found = i0 + __ffs(hit) - 1;
            }
            if (all >= need) break;
            need -= all;
        }
        __syncthreads();
        const Cut c{x, at_found};
        __syncthreads();
        return c;
    };
    if (!done) {
    if (ranks) cut = find_cut(cut, true, [](float) -> u64 { return 1; }, [&](u64) { return (u64)s.k; });
    if (s.p < 1.0) cut = find_cut(cut, false, weight, [&](u64 total) { return goal_of(s.p, total); });
    if (s.minw > 0.0) {
        const float x = weigh.min_p_cut(s.minw);
        int at = 0x7fffffff;
        if (s.minw > 1099511627776.0) {                // nothing weighs enough: the largest logit's lowest index stays
            if (tid == 0) at_found = 0x7fffffff;
            __syncthreads();
            each8([&](int c, const f8 &v) {
#pragma unroll
                for (int e = 0; e < 8; ++e) if (v[e] == m) atomicMin(&at_found, c + e);
            });
            __syncthreads();
            at = at_found;
        }
        if (x > cut.x) cut = Cut{x, at};
        else if (x == cut.x && at < cut.at) cut.at = at;
    }
    __syncthreads();
    // A wave's logits of one step of a pass lie in one piece.  Behind a cut few of them are kept: those are moved together in LDS, so that
    // 64 lanes weigh 64 kept logits.
    const bool all = cut.x == -INFINITY;
    float *q = queue[wave];
    if (SPLIT && !ranks && !(s.p < 1.0) && !(s.minw > 1099511627776.0)) for (int i = tid; i < pieces; i += NTHR) piece[i] = ws_row.piece[i];
    else each8([&](int i0, const f8 &v) {
        u64 sum = 0;
        if (all) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += weight(v[e]);
        } else {
            int n = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = inside(cut, v[e], i0 + e);
                const uint64_t b = __ballot(in);
                if (in) q[__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, n))] = v[e];
                n += __popcll(b);
            }
            wave_fence();
            for (int j = lane; j < n; j += 64) sum += weight(q[j]);
            wave_fence();
        }
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) piece[(i0 + 7) >> 9] = sum;
    });
    __syncthreads();
    }
    if (wave != 0) return;
    auto kept_weight = [&](float x, int i) -> u64 { return weight(inside(cut, x, i) ? x : -INFINITY); };
    u64 total = 0;
    for (int q = lane; q < pieces; q += 64) total += piece[q];
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    u64 t = point_of(a.u[row], total);
    int q0 = 0;
    for (;; q0 += 64) {                                // 64 pieces at a time
        const u64 one = q0 + lane < pieces ? piece[q0 + lane] : 0, inc = wave_scan(one);
        const u64 hit = __ballot(inc > t);
        if (hit) {
            const int w = __ffsll((long long)hit) - 1;
            t -= __shfl(inc - one, w, 64);
            q0 += w;
            break;
        }
        if (q0 + 64 >= pieces) break;                  // not reached: t < total
        t -= __shfl(inc, 63, 64);
    }
    const int i0 = q0 * 512 + lane * 8;
    u64 w8[8], sum = 0;
    {
        f8 v = splat8(-INFINITY);
        if (i0 < V) v = load8_n(l + i0, V - i0, -INFINITY);
#pragma unroll
        for (int e = 0; e < 8; ++e) { w8[e] = kept_weight(v[e], i0 + e); sum += w8[e]; }
    }
    const u64 inc = wave_scan(sum), hit = __ballot(inc > t);
    if (hit && lane == __ffsll((long long)hit) - 1) {
        u64 run = inc - sum;
        int e = 0;
        for (; e < 7; ++e) { run += w8[e]; if (run > t) break; }
        a.out[row] = i0 + e;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
namespace {
// Few long rows: maxima and weights are taken by many workgroups, one or two launches more.  In us, one workgroup per row and this, bf16
// rows of 128000: 1 row without a cut 41 and 17, with min-p 35 and 17, k = 50 21 and 15; 64 rows 43 and 25, 37 and 29, 23 and
// 17; 128 rows with min-p 38 and 45.  1 row of 65536 without a cut 24 and 16, of 40000 16 and 17.  Top-p alone: fp32 98 and 58,
// bf16, whose values are counted, 53 and 64.  Where the largest logit's index is all that is asked for: 10 and 14.
bool split_rows(const dnag_sample_args &p) {
    if (p.vocab < 65536 || p.vocab > SMP_MAX_V || p.rows < 1 || p.rows > 64 || p.top_k_rows || !(p.temperature_rows || p.temperature > 0.0)) return false;
    if (p.top_k > 0 && p.top_k < p.vocab) return p.top_k <= short_list_k(p.vocab, p.dtype == DNAG_BF16);
    return p.dtype != DNAG_BF16 || !(p.top_p_rows || p.top_p < 1.0);
}
int64_t space_of_row(int64_t V) { return (SMP_BINS * 8 + ws_pieces(V) * 8 + ws_groups(V) * 4 + 255) / 256 * 256; }

template <class T, bool SPLIT>
int launch_long(const SampleArgs &a, hipStream_t st) {
    const size_t bytes = (size_t)ws_pieces(a.V) * 8 + (__is_same(T, tbf16) ? 5120 * 8 : 0);      // pieces, and the slots' weights
    static LdsLimit limit;
    TOK_TRY(limit.allow((const void *)sample_row_kernel<T, 1024, SPLIT>, bytes, 52 * 1024));
    hipLaunchKernelGGL((sample_row_kernel<T, 1024, SPLIT>), dim3((unsigned)a.rows), dim3(1024), bytes, st, a);
    return 0;
}
template <class T>
int launch(const SampleArgs &a, hipStream_t st) {
    if (a.V <= 64) {
        const int G = pow2_at_least(a.V, 2, 64);
        hipLaunchKernelGGL((sample_small_kernel<T>), dim3((unsigned)ceil_div(a.rows, 256 / G)), dim3(256), 0, st, a, G);
    } else if (a.V <= 4096) {
        hipLaunchKernelGGL((sample_row_kernel<T, 256, false>), dim3((unsigned)a.rows), dim3(256), (size_t)ws_pieces(a.V) * 8, st, a);
    } else if (a.ws) {
        hipLaunchKernelGGL((sample_groups_kernel<T>), dim3((unsigned)ceil_div(a.V, 2048), (unsigned)a.rows), dim3(256), 0, st, a);
        if (!(a.top_k1 > 0 && a.top_k1 < a.V)) hipLaunchKernelGGL((sample_weights_kernel<T>), dim3((unsigned)ceil_div(a.V, 4096), (unsigned)a.rows), dim3(256), 0, st, a);
        if (int rc = launch_long<T, true>(a, st)) return rc;
    } else if (int rc = launch_long<T, false>(a, st)) return rc;
    TOK_TRY(hipGetLastError());
    return 0;
}
}  // namespace

extern "C" size_t dnag_sample_args_bytes(void) { return sizeof(dnag_sample_args); }

extern "C" size_t dnag_sample_workspace_bytes(const dnag_sample_args *p) {
    return p && split_rows(*p) ? (size_t)(p->rows * space_of_row(p->vocab)) : 0;
}

extern "C" int dnag_sample_tokens(const dnag_sample_args *p) {
    if (!p) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    if (!dtype_known(p->dtype)) return dnag_fail(DNAG_E_ARG, "unknown dtype %d", p->dtype);
    if (p->rows < 0 || p->rows > 0x7fffffffll) return dnag_fail(DNAG_E_ARG, "rows=%lld out of range", (long long)p->rows);
    if (p->vocab < 1 || p->vocab > SMP_MAX_V) return dnag_fail(DNAG_E_ARG, "vocab=%lld out of range (1 .. 2^20)", (long long)p->vocab);
    if (p->logits_stride < p->vocab) return dnag_fail(DNAG_E_ARG, "the logits' row stride %lld is smaller than vocab %lld", (long long)p->logits_stride, (long long)p->vocab);
    if (p->rows == 0) return 0;
    if (!p->logits || !p->u || !p->out) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    SampleArgs a = {};
    a.logits = p->logits; a.ld = p->logits_stride; a.rows = p->rows; a.V = (int)p->vocab;
    a.u = p->u; a.temperature = p->temperature_rows; a.top_p = p->top_p_rows; a.min_p = p->min_p_rows; a.top_k = p->top_k_rows;
    a.temperature1 = p->temperature; a.top_p1 = p->top_p; a.min_p1 = p->min_p; a.top_k1 = p->top_k;
    a.out = p->out;
    if (const size_t need = dnag_sample_workspace_bytes(p)) {
        if (!p->workspace || p->workspace_bytes < need) return dnag_fail(DNAG_E_WORKSPACE, "workspace has %zu bytes, %zu are needed", p->workspace_bytes, need);
        a.ws = (char *)p->workspace;
        a.ws_row = space_of_row(a.V);
    }
    hipStream_t st = (hipStream_t)p->stream;
    constexpr int64_t MOST = 1 << 21;                  // rows of a launch: 2^32 lanes are more than a grid holds
    const int64_t row_bytes = a.ld * (p->dtype == DNAG_F32 ? 4 : 2);
    while (a.rows > 0) {
        const int64_t left = a.rows - MOST;
        if (left > 0) a.rows = MOST;
        if (int rc = p->dtype == DNAG_F32 ? launch<float>(a, st) : p->dtype == DNAG_BF16 ? launch<tbf16>(a, st) : launch<tf16>(a, st)) return rc;
        a.logits = (const char *)a.logits + MOST * row_bytes;
        a.u += MOST;
        a.out += MOST;
        if (a.temperature) a.temperature += MOST;
        if (a.top_k) a.top_k += MOST;
        if (a.top_p) a.top_p += MOST;
        if (a.min_p) a.min_p += MOST;
        a.rows = left;
    }
    return 0;
}
