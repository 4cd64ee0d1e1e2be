// Distillation from a teacher's top logits.  Row t: q = softmax(s / tau) over the student's V logits, p = softmax(z / tau)
// over the teacher's K entries z with indices i_k (an index outside 0 .. V - 1 is no entry; indices may repeat):
//   loss_t = w_t tau^2 sum_k p_k (log p_k - log q_{i_k}),      d loss_t / d s_j = w_t tau (q_j - sum_{k: i_k = j} p_k)
// A row without entries or with a weight that is not positive gives 0 and gradients of 0 and its logits are not read.
//
// Bound by HBM: the loss reads T V logits, loss and gradient together read them once and write T V.  A team of TPR lanes
// keeps its row's raw elements in registers (NV pieces of eight per lane) between the maximum, the sum and the gradient;
// above 131072 16-bit or 65536 fp32 logits (NV = 0) the row is read again, out of the caches.  The teacher's entries are the first wave's work beside
// that; the few elements of the gradient that hold an entry are written again, in full precision, behind the row.
// Sums are fp32, in a fixed order.  Exponentials are v_exp_f32 (1 ulp) of s c - R, one fused operation, with c = log2(e) / tau and R the
// rounded c max(s): what its rounding takes from every exponent is one factor, taken out of the sum.
// 8192 x 32000 bf16, a tenth of the rows without weight, loss and gradient: 243 us, 4.1 TB/s; the loss alone 88 us, 5.4 TB/s; the gradient from its
// statistics 191 us, 5.2 TB/s.  1000 x 50001 fp16, loss: 32 us, 2.8 TB/s: rows of odd length are read by 2-byte-aligned vector loads, and a CU holds two of the 13-wave workgroups
// at a time, so that 1000 take two rounds.  More than a hundred entries cost their search for equal indices, k^2 / 64 steps of one wave for each
// row: loss and gradient with k = 256 513 us, with k = 1024 4.9 ms (the loss alone 277 us).  16 pieces of 16-bit logits (from 65537 to 131072)
// leave up to 584 bytes a lane in scratch: 2048 x 128000 bf16 618 us, 1.6 TB/s.
#include "dnag_token_common.h"
#include <math.h>

#define DISTILL_MAX_K 1024

struct DistillArgs {
    const void *logits, *tids, *tlogits;
    int64_t ld, rows;
    int V, K, ids8, tdtype, mean;
    float tau, c2;                                     // c2 = log2(e) / tau
    const float *weight;                               // [rows] or NULL
    const float *wsum;                                 // sum of the positive weights (mean with weights) or NULL
    float scale;                                       // 1 / rows (mean without weights) or 1
    float *row_loss;                                   // [rows] or NULL: w_t tau^2 KL_t
    float *stats;                                      // [rows][2] or NULL: largest logit, sum of exponentials relative to it
    const float *gout;                                 // MODE 2: upstream gradient, gout[t * gstep]
    int64_t gstep;
    void *grad;
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// MODE 0: loss (and stats), 1: loss and gradient, 2: gradient from stats and the upstream gradient
template <class T, int TPR, int NV, int MODE>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void distill_kernel
(const DistillArgs a) {
    constexpr int NT = TPR <= 64 ? 256 / TPR : 1, TW = TPR < 64 ? TPR : 64;      // TW: lanes that handle the teacher's entries
    constexpr int NR = NV > 0 ? NV : 1;
    constexpr float LOW = __is_same(T, tf16) ? -65536.f : -3.402823466e38f;      // no finite logit is below: -inf - LOW = -inf, exp2 = 0
    typedef typename Vec8<T>::type raw8;
    extern __shared__ char lds[];
    __shared__ float red[33];                          // pairs of the waves; [32]: the teacher's maximum
    float *tp = (float *)lds + (size_t)(TPR > 64 ? 0 : threadIdx.x / TPR) * 3 * a.K;      // the team's entries: teacher's logit, index, student's logit
    int *ti = (int *)(tp + a.K);
    float *ts = tp + 2 * a.K;
    // a team above 64 lanes is the workgroup, which has as many waves as the row needs
    const int tpr = TPR > 64 ? (int)blockDim.x : TPR, lane = TPR > 64 ? threadIdx.x : threadIdx.x & (TPR - 1);
    const int64_t row = (int64_t)blockIdx.x * NT + (TPR > 64 ? 0 : threadIdx.x / TPR);
    if (row >= a.rows) return;
    const T *s = (const T *)a.logits + row * a.ld;
    T *g = MODE > 0 ? (T *)a.grad + row * a.V : nullptr;
    const float w = a.weight ? a.weight[row] : 1.f;
    const bool on = w > 0.f;
    auto zero_row = [&]() {
        if constexpr (MODE > 0)
            for (int c = lane * 8; c < a.V; c += tpr * 8) store8_n(g + c, splat8(0.f), a.V - c);
        if (MODE < 2 && lane == 0) {
            if (a.row_loss) a.row_loss[row] = 0.f;
            if (a.stats) { a.stats[2 * row] = 0.f; a.stats[2 * row + 1] = 1.f; }
        }
    };
    if (!on) { zero_row(); return; }                   // the same for the whole team
    // the row, raw, issued before anything waits
    raw8 x[NR];
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + lane) * 8, n = a.V - c;
            if (n >= 8) x[j] = load8_raw(s + c);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = e < n ? s[c + e] : (T)(-INFINITY);
        }
    }
    // the teacher: the first TW lanes of the team
    float tmax = -INFINITY, tsum = 0.f;
    if (lane < TW) {
        for (int k = lane; k < a.K; k += TW) {
            const size_t at = (size_t)row * a.K + k;
            const int64_t i = a.ids8 ? ((const int64_t *)a.tids)[at] : (int64_t)((const int32_t *)a.tids)[at];
            const bool in = i >= 0 && i < a.V;
            const float z = a.tdtype == DNAG_F32 ? ((const float *)a.tlogits)[at] : a.tdtype == DNAG_BF16 ? (float)((const tbf16 *)a.tlogits)[at]
                                                                                                          : (float)((const tf16 *)a.tlogits)[at];
            tp[k] = in ? z : -INFINITY;
            ti[k] = in ? (int)i : -1;
            ts[k] = in ? (float)s[i] : 0.f;
            if (in) tmax = z != z || tmax != tmax ? NAN : fmaxf(tmax, z);          // a NaN among the entries stays one
        }
#pragma unroll
        for (int o = TW / 2; o > 0; o >>= 1) { const float b = __shfl_xor(tmax, o, 64); tmax = tmax != tmax || b != b ? NAN : fmaxf(tmax, b); }
        if (tmax != -INFINITY) {
            for (int k = lane; k < a.K; k += TW) tsum += exp2_hw((tp[k] - tmax) * a.c2);
#pragma unroll
            for (int o = TW / 2; o > 0; o >>= 1) tsum += __shfl_xor(tsum, o, 64);
        }
        if constexpr (TPR > 64) if (lane == 0) red[32] = tmax;
    }
    if constexpr (TPR > 64) { __syncthreads(); tmax = red[32]; }
    if (tmax == -INFINITY) { zero_row(); return; }     // no entry (the same for the whole team)
    // Every lane takes its exponentials relative to its own reference `tr`, in fp32 (MODE 1 keeps them for the gradient), so that one
    // exchange of (reference, sum) pairs gives the row's.
    constexpr bool KEEP = MODE == 1 && NV > 0 && NV <= 8;      // 16 pieces: their registers would spill
    float ref, sum, tr = LOW, own = 0.f;
    f8 ex[KEEP ? NV : 1];
    // exp((x - r) / tau) times 2^(r c - R) for R the rounded r c, a power near 1 that `true_to` takes out; where the reference is so large that
    // it is not near 1 (a mask's values all over a row), from the difference
    // (fp16 cannot get there from a temperature of 0.1 on, the least that is built for it: the difference and its registers cost the loss of
    // 1000 x 50001 38 us for 32)
    auto far = [&](float r) { return __is_same(T, tf16) ? false : !(fabsf(r * a.c2) < 1048576.f); };
    auto exps = [&](f8 v, float r) {                   // (without a branch: two forms of it took 6 % longer)
        const float base = far(r) ? r : 0.f, R = far(r) ? 0.f : r * a.c2;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = exp2_hw(fmaf(v[e] - base, a.c2, -R));
        return v;
    };
    auto true_to = [&](float r) { return far(r) ? 1.f : exp2_hw(-fmaf(r, a.c2, -(r * a.c2))); };
    auto shift = [&](float from, float to) { return exp2_hw((from - to) * a.c2); };
    if constexpr (MODE == 2) { ref = a.stats[2 * row]; sum = a.stats[2 * row + 1]; }
    else {
        if constexpr (NV > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j) tr = fmaxf(tr, max8(widen<T>(x[j])));
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const f8 v = exps(widen<T>(x[j]), tr);
                own += sum8(v);
                if constexpr (KEEP) ex[j] = v;
            }
            own *= true_to(tr);
        } else
            for (int c = lane * 8; c < a.V; c += tpr * 8) {
                const f8 v = load8_n(s + c, a.V - c, -INFINITY);
                const float nr = fmaxf(tr, max8(v));
                own *= shift(tr, nr);
                tr = nr;
                own += sum8(exps(v, tr)) * true_to(tr);
            }
        ref = tr;
#pragma unroll
        for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor(ref, o, 64));
        sum = own * shift(tr, ref);
#pragma unroll
        for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if constexpr (TPR > 64) {
            if ((threadIdx.x & 63) == 0) { red[2 * (threadIdx.x >> 6)] = ref; red[2 * (threadIdx.x >> 6) + 1] = sum; }
            __syncthreads();
            const int waves = tpr >> 6;
            for (int w = 0; w < waves; ++w) ref = fmaxf(ref, red[2 * w]);
            sum = 0.f;
            for (int w = 0; w < waves; ++w) sum += red[2 * w + 1] * shift(red[2 * w], ref);
        }
    }
    if constexpr (MODE < 2) {
        if (lane < TW) {
            const float ltsum = log2f(tsum), lsum = log2f(sum);
            float l = 0.f;
            for (int k = lane; k < a.K; k += TW) {
                if (ti[k] < 0) continue;
                const float u = (tp[k] - tmax) * a.c2, p = exp2_hw(u) / tsum;
                if (!(p == 0.f)) l += p * ((u - ltsum) - ((ts[k] - ref) * a.c2 - lsum));
            }
#pragma unroll
            for (int o = TW / 2; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
            if (lane == 0) {
                if (a.row_loss) a.row_loss[row] = a.tau * a.tau * w * (l * 0.69314718056f);
                if (a.stats) { a.stats[2 * row] = ref; a.stats[2 * row + 1] = sum; }
            }
        }
    }
    if constexpr (MODE > 0) {
        float f = w * a.tau * a.scale;
        if (a.wsum) f /= *a.wsum;                      // positive: this row's weight is part of it
        if constexpr (MODE == 2) f *= a.gout[row * a.gstep];
        const float fq = f / sum;
        const float ft = fq * (KEEP ? true_to(tr) * shift(tr, ref) : true_to(ref));
        if constexpr (KEEP) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * tpr + lane) * 8;
                if (c < a.V) store8_n(g + c, ex[j] * ft, a.V - c);
            }
        } else if constexpr (NV > 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * tpr + lane) * 8;
                if (c < a.V) store8_n(g + c, exps(widen<T>(x[j]), ref) * ft, a.V - c);
            }
        } else
            for (int c = lane * 8; c < a.V; c += tpr * 8) store8_n(g + c, exps(load8_n(s + c, a.V - c), ref) * ft, a.V - c);
        if constexpr (TPR > 64) __syncthreads();       // the row is written before its entries are
        else wave_fence();
        if (lane < TW)
            for (int k = lane; k < a.K; k += TW) {
                const int i = ti[k];
                if (i < 0) continue;
                float z = 0.f;
                bool first = true;
                for (int j = 0; j < a.K; ++j)
                    if (ti[j] == i) { z += exp2_hw((tp[j] - tmax) * a.c2); first &= j >= k; }
                if (first) g[i] = (T)(f * (shift(ts[k], ref) / sum - z / tsum));
            }
    }
}

// sum of the positive weights, one block, fixed order
__global__ __launch_bounds__(1024) void distill_weight_kernel(const float *__restrict__ w, int64_t rows, float *__restrict__ out) {
    __shared__ float q[16];
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < rows; i += 8192) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) { const int64_t q = i + u * 1024; x[u] = w[q < rows ? q : i]; if (!(q < rows && x[u] > 0.f)) x[u] = 0.f; }
#pragma unroll
        for (int u = 0; u < 8; ++u) s += x[u];
    }
    s = team_sum<64>(s);
    if ((threadIdx.x & 63) == 0) q[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) s += q[k];
        *out = s;
    }
}
__global__ __launch_bounds__(1024) void distill_loss_kernel(const float *__restrict__ row_loss, int64_t rows, const float *__restrict__ wsum, float scale,
                                                            float *__restrict__ out) {
    __shared__ float q[16];
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < rows; i += 8192) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) { const int64_t q = i + u * 1024; x[u] = row_loss[q < rows ? q : i]; }
#pragma unroll
        for (int u = 0; u < 8; ++u) s += i + u * 1024 < rows ? x[u] : 0.f;
    }
    s = team_sum<64>(s);
    if ((threadIdx.x & 63) == 0) q[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) s += q[k];
        *out = wsum ? (*wsum > 0.f ? s / *wsum : 0.f) : s * scale;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
namespace {
int check(const dnag_distill_args *p) {
    if (!p) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    if (!dtype_known(p->dtype) || !dtype_known(p->teacher_dtype)) return dnag_fail(DNAG_E_ARG, "unknown dtype %d / %d", p->dtype, p->teacher_dtype);
    if (p->ids_bytes != 4 && p->ids_bytes != 8) return dnag_fail(DNAG_E_ARG, "teacher ids of %d bytes (4 or 8 are built)", p->ids_bytes);
    if (p->rows < 0 || p->rows > 0x7fffffffll) return dnag_fail(DNAG_E_ARG, "rows=%lld out of range", (long long)p->rows);
    if (p->vocab < 1 || p->vocab > (1 << 30)) return dnag_fail(DNAG_E_ARG, "vocab=%lld out of range (1 .. 2^30)", (long long)p->vocab);
    if (p->k < 1 || p->k > DISTILL_MAX_K) return dnag_fail(DNAG_E_ARG, "k=%d out of range (1 .. %d)", p->k, DISTILL_MAX_K);
    const float least = p->dtype == DNAG_F16 ? 0.1f : 1e-6f;
    if (!(p->temperature >= least && p->temperature <= 1e6f)) return dnag_fail(DNAG_E_ARG, "temperature=%g out of range (%g .. 1e6)", (double)p->temperature, (double)least);
    if (p->logits_stride < p->vocab) return dnag_fail(DNAG_E_ARG, "the logits' row stride %lld is smaller than vocab %lld", (long long)p->logits_stride, (long long)p->vocab);
    if (p->reduction < DNAG_REDUCE_NONE || p->reduction > DNAG_REDUCE_MEAN) return dnag_fail(DNAG_E_ARG, "unknown reduction %d", p->reduction);
    return 0;
}
struct Ws { size_t wsum, row_loss, bytes; };
Ws plan(const dnag_distill_args &p) {
    Ws w;
    w.wsum = 0;
    w.row_loss = 256;
    w.bytes = 256 + (p.reduction == DNAG_REDUCE_NONE ? 0 : align256((size_t)p.rows * 4));
    return w;
}
DistillArgs fill(const dnag_distill_args &p) {
    DistillArgs a = {};
    a.logits = p.logits; a.tids = p.teacher_ids; a.tlogits = p.teacher_logits;
    a.ld = p.logits_stride; a.rows = p.rows;
    a.V = (int)p.vocab; a.K = p.k; a.ids8 = p.ids_bytes == 8; a.tdtype = p.teacher_dtype;
    a.tau = p.temperature; a.c2 = (float)(1.4426950408889634 / (double)p.temperature);
    a.weight = p.row_weight;
    const bool mean = p.reduction == DNAG_REDUCE_MEAN;
    a.wsum = mean && p.row_weight ? (const float *)p.workspace : nullptr;
    a.scale = mean && !p.row_weight ? 1.0f / (float)p.rows : 1.0f;
    return a;
}
int weights(const DistillArgs &a, float *wsum, hipStream_t st) {
    if (!a.wsum) return 0;
    hipLaunchKernelGGL(distill_weight_kernel, dim3(1), dim3(1024), 0, st, a.weight, a.rows, wsum);
    TOK_TRY(hipGetLastError());
    return 0;
}
template <class T, int MODE, int TPR, int NV>
int launch(const DistillArgs &a, float *wsum, hipStream_t st) {
    constexpr int NT = TPR <= 64 ? 256 / TPR : 1;
    const int64_t lanes = NV > 0 ? ceil_div(a.V, 8 * NV) : TPR;        // a team above 64 lanes: whole waves, as many as the row fills
    const unsigned threads = TPR <= 64 ? 256 : (unsigned)(ceil_div(lanes, 64) * 64);
    if (int rc = grid_fits(ceil_div(a.rows, NT), threads)) return rc;
    if (int rc = weights(a, wsum, st)) return rc;      // the call's first launch: nothing is refused behind it
    hipLaunchKernelGGL((distill_kernel<T, TPR, NV, MODE>), dim3((unsigned)ceil_div(a.rows, NT)), dim3(threads), (size_t)NT * a.K * 12, st, a);
    TOK_TRY(hipGetLastError());
    return 0;
}
// lanes of a row's team and pieces of eight elements that a lane keeps: the smallest team that holds the row
template <class T, int MODE>
int launch_size(const DistillArgs &a, float *wsum, hipStream_t st) {
    const int V = a.V;
    if (V <= 64 && a.K <= 128) return launch<T, MODE, 8, 1>(a, wsum, st);
    if (V <= 512) return launch<T, MODE, 64, 1>(a, wsum, st);
    if (V <= 2048) return launch<T, MODE, 64, 4>(a, wsum, st);
    if (V <= 8192) return launch<T, MODE, 256, 4>(a, wsum, st);
    if (V <= 32768) return launch<T, MODE, 512, 8>(a, wsum, st);
    if (V <= 65536) return launch<T, MODE, 1024, 8>(a, wsum, st);
    if (sizeof(T) == 2 && V <= 131072) return launch<T, MODE, 1024, sizeof(T) == 2 ? 16 : 0>(a, wsum, st);
    return launch<T, MODE, 1024, 0>(a, wsum, st);
}
template <int MODE>
int launch_type(int dtype, const DistillArgs &a, float *wsum, hipStream_t st) {
    return dtype == DNAG_F32 ? launch_size<float, MODE>(a, wsum, st) : dtype == DNAG_BF16 ? launch_size<tbf16, MODE>(a, wsum, st) : launch_size<tf16, MODE>(a, wsum, st);
}
int forward(const dnag_distill_args *p, bool with_grad) {
    if (int rc = check(p)) return rc;
    if (p->rows == 0) return dnag_fail(DNAG_E_ARG, "no rows: the loss is 0, nothing is launched");
    if (!p->logits || !p->teacher_ids || !p->teacher_logits || !p->loss || (with_grad && !p->grad)) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    const Ws w = plan(*p);
    if (!p->workspace || p->workspace_bytes < w.bytes) return dnag_fail(DNAG_E_WORKSPACE, "workspace has %zu bytes, %zu are needed", p->workspace_bytes, w.bytes);
    hipStream_t st = (hipStream_t)p->stream;
    DistillArgs a = fill(*p);
    const bool none = p->reduction == DNAG_REDUCE_NONE;
    a.row_loss = none ? p->loss : (float *)((char *)p->workspace + w.row_loss);
    a.stats = p->stats;
    a.grad = p->grad;
    float *wsum = (float *)p->workspace;
    if (int rc = with_grad ? launch_type<1>(p->dtype, a, wsum, st) : launch_type<0>(p->dtype, a, wsum, st)) return rc;
    if (!none) {
        hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, st, a.row_loss, p->rows, a.wsum, a.scale, p->loss);
        TOK_TRY(hipGetLastError());
    }
    return 0;
}
}  // namespace

extern "C" size_t dnag_distill_args_bytes(void) { return sizeof(dnag_distill_args); }
extern "C" size_t dnag_distill_workspace_bytes(const dnag_distill_args *p) { return check(p) ? 0 : plan(*p).bytes; }
extern "C" int dnag_distill_loss(const dnag_distill_args *p) { return forward(p, false); }
extern "C" int dnag_distill_loss_grad(const dnag_distill_args *p) { return forward(p, true); }

extern "C" int dnag_distill_backward(const dnag_distill_args *p) {
    if (int rc = check(p)) return rc;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->teacher_ids || !p->teacher_logits || !p->stats || !p->grad_out || !p->grad) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    const Ws w = plan(*p);
    if (!p->workspace || p->workspace_bytes < w.bytes) return dnag_fail(DNAG_E_WORKSPACE, "workspace has %zu bytes, %zu are needed", p->workspace_bytes, w.bytes);
    DistillArgs a = fill(*p);
    a.stats = p->stats;
    a.gout = p->grad_out;
    a.gstep = p->reduction == DNAG_REDUCE_NONE ? 1 : 0;
    a.grad = p->grad;
    return launch_type<2>(p->dtype, a, (float *)p->workspace, (hipStream_t)p->stream);
}
