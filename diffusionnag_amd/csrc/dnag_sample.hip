// Drawing one token per row of logits with temperature, top-k, top-p and min-p from given uniform numbers.
//   weights    e_i = exp((l_i - max l) / T), held as whole numbers w_i = round(2^40 e_i)
//   top-k      the k largest logits; equal logits in the order of their index
//   top-p      of those, the shortest run of largest ones whose weights reach p times their sum (at least one)
//   min-p      of those, the ones with e_i >= min_p (the largest always)
//   token      the first index, in index order, whose running sum of kept weights exceeds u times their total
// T <= 0: the largest logit's lowest index.  NaN and -inf are never drawn; a row of nothing else gives -1.
//
// Whole-number weights make every sum independent of its order (LDS atomics among them) and every comparison exact: the
// token is a function of the row, whichever threads it falls to.  exp is fp64 (an fp32 one moves the border between two
// tokens by 1e-7, which over a flat row of 10^5 tokens changes one draw in a few hundred); 2^-40 is below what a uniform
// fp32 number resolves.  A cut (top-k, top-p) is found by histograms: 2048 equal steps of (max - l) / T, then, inside the step where the
// sum passes its goal, eleven, eleven and ten bits of the logit's ordered bit pattern, then the index among equal logits.
// One workgroup per row, the row read again (out of the caches) by each pass; rows of at most 64 logits take a team of
// lanes each and rank by comparing all pairs.
#include "dnag_token_common.h"
#include <math.h>

#define SMP_BINS 2048
#define SMP_RANGE 28.0f          // exp(-28) < 2^-40: weights beyond are 0
#define SMP_ONE 1099511627776.0  // 2^40
#define SMP_MAX_V (1 << 20)      // sums stay below 2^60

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
};
struct RowSet { double it, p, minp; int k; bool greedy; };
__device__ __forceinline__ RowSet row_set(const SampleArgs &a, int64_t row) {
    RowSet s;
    const double t = a.temperature ? (double)a.temperature[row] : a.temperature1;
    s.greedy = !(t > 0.0);
    s.it = 1.0 / t;
    s.p = a.top_p ? (double)a.top_p[row] : a.top_p1;
    s.minp = a.min_p ? (double)a.min_p[row] : a.min_p1;
    if (s.minp != s.minp) s.minp = 0.0;
    s.k = a.top_k ? a.top_k[row] : a.top_k1;
    return s;
}
// a logit as compared: NaN counts as -inf, -0 as +0
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
// order of the bit patterns = order of the values
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ double raw_weight(float x, float m, double it) { return x == m ? 1.0 : exp(((double)x - (double)m) * it); }
__device__ __forceinline__ u64 whole_weight(double e) { return (u64)rint(e * SMP_ONE); }
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
            const double e = live ? raw_weight(x, m, s.it) : 0.0;
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
            kept = kept && (e >= s.minp || rank == 0);
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

// ---- one workgroup per row -----------------------------------------------------------------------------------------------
struct Cut {                       // kept: in an earlier step, or in this one with a larger key, or an equal key and index <= at
    int step;
    uint32_t key;
    int at;
};
template <class T, int NTHR>
__global__ __launch_bounds__(NTHR) void sample_row_kernel(const SampleArgs a) {
    constexpr int NW = NTHR / 64, PER = SMP_BINS / NTHR;
    extern __shared__ u64 piece[];                     // sums of 512 logits each, for the draw
    __shared__ u64 hist[SMP_BINS];
    __shared__ u64 ws[NW];
    __shared__ float wf[NW];
    __shared__ u64 found[3];                           // bin, sum before it, sum in it
    __shared__ int at_found;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const T *l = (const T *)a.logits + row * a.ld;
    const int V = a.V;
    const RowSet s = row_set(a, row);
    auto each8 = [&](auto f) {                         // f(first index, eight cleaned logits); -inf past the end
        for (int c = tid * 8; c < V; c += NTHR * 8) {
            f8 v = load8_n(l + c, V - c, -INFINITY);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = clean(v[e]);
            f(c, v);
        }
    };
    float m = -INFINITY;
    each8([&](int, const f8 &v) { m = fmaxf(m, max8(v)); });
    m = team_max<64>(m);
    if (lane == 0) wf[wave] = m;
    if (tid == 0) at_found = 0x7fffffff;
    __syncthreads();
    for (int w = 0; w < NW; ++w) m = fmaxf(m, wf[w]);
    if (m == -INFINITY) { if (tid == 0) a.out[row] = -1; return; }
    if (s.greedy) {
        int first = 0x7fffffff;
        each8([&](int c, const f8 &v) {
#pragma unroll
            for (int e = 7; e >= 0; --e) if (v[e] == m && c + e < first) first = c + e;
        });
        if (first != 0x7fffffff) atomicMin(&at_found, first);
        __syncthreads();
        if (tid == 0) a.out[row] = at_found;
        return;
    }
    const float per_step = (float)(s.it * (double)(SMP_BINS / SMP_RANGE));
    auto step_of = [&](float x) -> int {               // never falls as x falls
        if (x == m) return 0;
        const float q = (m - x) * per_step;
        return q < (float)(SMP_BINS - 1) ? (int)q : SMP_BINS - 1;
    };
    auto weight = [&](float x) -> u64 {
        if (x != m && ((double)x - (double)m) * s.it < -(double)SMP_RANGE) return 0;
        return whole_weight(raw_weight(x, m, s.it));
    };
    auto inside = [&](const Cut &c, float x, int i) {
        const int b = step_of(x);
        if (b != c.step) return b < c.step;
        const uint32_t k = ordered(x);
        return k > c.key || (k == c.key && i <= c.at);
    };
    auto clear = [&]() {
        __syncthreads();
        for (int b = tid; b < SMP_BINS; b += NTHR) hist[b] = 0;
        __syncthreads();
    };
    // the first bin whose running sum reaches the goal; goal(total) is asked once the total is known
    auto scan = [&](auto goal) {
        __syncthreads();
        u64 h[PER], sum = 0;
#pragma unroll
        for (int q = 0; q < PER; ++q) { h[q] = hist[tid * PER + q]; sum += h[q]; }
        u64 inc = sum;
        for (int o = 1; o < 64; o <<= 1) { const u64 b = __shfl_up(inc, o, 64); if (lane >= o) inc += b; }
        if (lane == 63) ws[wave] = inc;
        if (tid == 0) found[0] = SMP_BINS;
        __syncthreads();
        u64 total = 0, before = inc - sum;
        for (int w = 0; w < NW; ++w) { if (w < wave) before += ws[w]; total += ws[w]; }
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
    auto find_cut = [&](auto was, auto wt, auto goal) {
        Cut c{SMP_BINS, 0, -1};                        // everything
        clear();
        each8([&](int i0, const f8 &v) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[e] > -INFINITY && was(v[e], i0 + e)) {
                    const u64 w = wt(v[e]);
                    if (w) atomicAdd(&hist[step_of(v[e])], w);
                }
        });
        u64 want = scan(goal);
        if (found[0] == SMP_BINS) return c;            // the goal is not reached: all are kept
        c.step = (int)found[0];
        uint32_t prefix = 0;
        for (int shift = 21; found[2] != want - found[1]; shift = shift == 21 ? 10 : 0) {
            const int bits = shift == 0 ? 10 : 11;
            want -= found[1];
            clear();
            each8([&](int i0, const f8 &v) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (v[e] > -INFINITY && step_of(v[e]) == c.step && was(v[e], i0 + e)) {
                        const uint32_t k = ordered(v[e]);
                        if (shift == 21 || (k >> (shift + bits)) == prefix)
                            atomicAdd(&hist[(1 << bits) - 1 - ((k >> shift) & ((1u << bits) - 1))], wt(v[e]));
                    }
            });
            scan([&](u64) { return want; });
            prefix = (prefix << bits) | ((1u << bits) - 1 - (uint32_t)found[0]);
            c.key = shift ? (prefix << shift) - 1 : prefix;             // while the loop ends here: every key of the prefix is kept
            if (shift == 0) {
                // equal logits: as many as it takes, by index
                if (found[2] == want - found[1]) { c.at = 0x7fffffff; break; }
                const float x = __uint_as_float(c.key ^ (c.key & 0x80000000u ? 0x80000000u : 0xffffffffu));
                const u64 w1 = wt(x);
                u64 need = (want - found[1] + w1 - 1) / w1;             // the need-th of them is the last one kept
                for (int c0 = 0; c0 < V; c0 += NTHR * 8) {
                    const int i0 = c0 + tid * 8;
                    uint32_t hit = 0;
                    if (i0 < V) {
                        const f8 v = load8_n(l + i0, V - i0, -INFINITY);
#pragma unroll
                        for (int e = 0; e < 8; ++e) { const float y = clean(v[e]); if (y == x && was(y, i0 + e)) hit |= 1u << e; }
                    }
                    u64 n = __popc(hit), inc = n;
                    for (int o = 1; o < 64; o <<= 1) { const u64 b = __shfl_up(inc, o, 64); if (lane >= o) inc += b; }
                    __syncthreads();
                    if (lane == 63) ws[wave] = inc;
                    __syncthreads();
                    u64 before = inc - n, all = 0;
                    for (int w = 0; w < NW; ++w) { if (w < wave) before += ws[w]; all += ws[w]; }
                    if (before < need && before + n >= need) {
                        for (u64 q = before + 1; q < need; ++q) hit &= hit - 1;
                        at_found = i0 + __ffs(hit) - 1;
                    }
                    if (all >= need) break;
                    need -= all;
                }
                __syncthreads();
                c.at = at_found;
                break;
            }
        }
        __syncthreads();
        return c;
    };
    Cut ck{SMP_BINS, 0, -1}, cp{SMP_BINS, 0, -1};
    if (s.k > 0 && s.k < V) ck = find_cut([](float, int) { return true; }, [](float) -> u64 { return 1; }, [&](u64) { return (u64)s.k; });
    if (s.p < 1.0) cp = find_cut([&](float x, int i) { return inside(ck, x, i); }, weight, [&](u64 total) { return goal_of(s.p, total); });
    // the largest logit's lowest index is kept whatever min_p is
    int top = -1;
    if (s.minp > 1.0) {
        if (tid == 0) at_found = 0x7fffffff;
        __syncthreads();
        each8([&](int c, const f8 &v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) if (v[e] == m) atomicMin(&at_found, c + e);
        });
        __syncthreads();
        top = at_found;
    }
    auto kept_weight = [&](float x, int i) -> u64 {
        if (!(x > -INFINITY) || !inside(ck, x, i) || !inside(cp, x, i)) return 0;
        if (x != m && ((double)x - (double)m) * s.it < -(double)SMP_RANGE) return 0;
        const double e = raw_weight(x, m, s.it);
        return e >= s.minp || i == top ? whole_weight(e) : 0;
    };
    const int pieces = (V + 511) / 512;
    __syncthreads();
    for (int q = wave; q < pieces; q += NW) {          // the wave's pieces of 512 logits
        const int i0 = q * 512 + lane * 8;
        u64 sum = 0;
        if (i0 < V) {
            const f8 v = load8_n(l + i0, V - i0, -INFINITY);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += kept_weight(clean(v[e]), i0 + e);
        }
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) piece[q] = sum;
    }
    __syncthreads();
    if (wave != 0) return;
    u64 total = 0;
    for (int q = lane; q < pieces; q += 64) total += piece[q];
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    u64 t = point_of(a.u[row], total);
    int q0 = 0;
    for (;; q0 += 64) {                                // 64 pieces at a time
        u64 inc = q0 + lane < pieces ? piece[q0 + lane] : 0;
        const u64 one = inc;
        for (int o = 1; o < 64; o <<= 1) { const u64 b = __shfl_up(inc, o, 64); if (lane >= o) inc += b; }
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
        for (int e = 0; e < 8; ++e) { w8[e] = i0 + e < V ? kept_weight(clean(v[e]), i0 + e) : 0; sum += w8[e]; }
    }
    u64 inc = sum;
    for (int o = 1; o < 64; o <<= 1) { const u64 b = __shfl_up(inc, o, 64); if (lane >= o) inc += b; }
    const u64 hit = __ballot(inc > t);
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
template <class T>
int launch(const SampleArgs &a, hipStream_t st) {
    if (a.V <= 64) {
        const int G = pow2_at_least(a.V, 2, 64);
        hipLaunchKernelGGL((sample_small_kernel<T>), dim3((unsigned)ceil_div(a.rows, 256 / G)), dim3(256), 0, st, a, G);
    } else if (a.V <= 4096) {
        hipLaunchKernelGGL((sample_row_kernel<T, 256>), dim3((unsigned)a.rows), dim3(256), (size_t)ceil_div(a.V, 512) * 8, st, a);
    } else {
        hipLaunchKernelGGL((sample_row_kernel<T, 1024>), dim3((unsigned)a.rows), dim3(1024), (size_t)ceil_div(a.V, 512) * 8, st, a);
    }
    TOK_TRY(hipGetLastError());
    return 0;
}
}  // namespace

extern "C" size_t dnag_sample_args_bytes(void) { return sizeof(dnag_sample_args); }

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
    hipStream_t st = (hipStream_t)p->stream;
    return p->dtype == DNAG_F32 ? launch<float>(a, st) : p->dtype == DNAG_BF16 ? launch<tbf16>(a, st) : launch<tf16>(a, st);
}
