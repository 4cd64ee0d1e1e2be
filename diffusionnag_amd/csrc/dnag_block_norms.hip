// The seam between two blocks of a network: the norm behind a block with the block's gate and the residual scale, and the
// norm in front of the next block, in one pass over the rows.
//   forward:   x' = rs x + g N_post(y),   h = N_pre(x')          (y == NULL: h = N_pre(x), the entry of the first block)
//   N is RMSNorm (v / rms(v) w) or LayerNorm ((v - mean) / std w + b); g is one row for every `rows_per_gate` rows.
//   backward:  with a = dh w_pre, xhat = (x' - mean) r:   d = dx' + r (a - [mean a] - xhat mean(a xhat)),   dx = rs d,
//              dg += d n,  b = d g w_post,  dy = r_y (b - [mean b] - yhat mean(b yhat)),  dw += rows' sums    ([.]: LayerNorm)
//   The backward pass reads x and y again and recomputes x' in fp32: as many bytes as reading a saved x', without its rounding.
// Bound by HBM: four rows per row forward, six or seven backward.  A team of TPR lanes holds a row in registers, eight
// columns per lane (and twice that above 8192 columns), so every value is read once; statistics are fp32 and two-pass
// (mean first) for LayerNorm.  16384 x 4096 bf16 forward: 99 us, 5.4 TB/s; backward 16384 x 2048 with fp32 rows beside bf16: 135 us,
// 4.5 TB/s.  Rows of more than 8192 columns keep their pieces and sums partly in scratch in the backward pass (the 128 registers of a lane
// of 1024 do not hold two pieces of each; 400 to 750 bytes a lane): 2048 x 16384 bf16 takes 372 us, its 403 MB at the copy rate 79.
// Gradients of the weights and of shared gates are summed by every block over its own rows in
// registers, then over blocks in block order by a second launch: no atomics, the same bits every time.
#include "dnag_token_common.h"

struct BnArgs {
    const void *x, *y, *gate, *pw, *pb, *qw, *qb;      // q*: the norm in front (pre), p*: the norm behind (post)
    void *xn, *h;
    const void *gx, *gh;                               // backward: gradients of xn and h
    void *dx, *dy, *dgate;
    float *part, *gpart;                               // backward: [blocks][arrays][d], [G][S][d]
    int64_t xs, ys, gxs, ghs;                          // row strides in elements
    int64_t rows, rpg, G;                              // rows per gate row, gate rows
    int64_t split_rows;                                // backward: rows of one work item (a gate row has S items)
    int S, d, pre, small32;                            // small32: bit 0 gate, bit 1 post norm, bit 2 pre norm are fp32
    int cell;                                          // backward, rpg < teams of a block: teams that share a run of rows (a power of two, within a wave)
    float rs, eps, inv_d;
};

template <int TPR> struct RowSum {
    float (*red)[16];
    int turn = 0;
    __device__ __forceinline__ float operator()(float v) {
        if constexpr (TPR <= 64) return team_sum<TPR>(v);
        v = team_sum<64>(v);
        float *b = red[turn];
        turn ^= 1;                                     // two buffers: the one being read is written again a barrier later
        if ((threadIdx.x & 63) == 0) b[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = b[0];
        const int waves = blockDim.x >> 6;             // as many as the row needs
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) s += w < waves ? b[w] : 0.f;
        return s;
    }
};

// v -> (v - mean) r in place; r returned.  Columns past d hold zeros and stay zeros.
template <bool LN, int NV, class Sum>
__device__ __forceinline__ float normalise(f8 (&v)[NV], const int (&n)[NV], Sum &sum, float eps, float inv_d) {
    if constexpr (LN) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) s += sum8(v[j]);
        const float mean = sum(s) * inv_d;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = e < n[j] ? v[j][e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) q += sum8(v[j] * v[j]);
    const float r = 1.0f / sqrtf(sum(q) * inv_d + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] *= r;
    return r;
}

template <class TX, class TY, int TPR, int NV, bool LN>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void block_norms_kernel(const BnArgs a) {
    constexpr int NT = TPR <= 64 ? 256 / TPR : 1;
    __shared__ float red[2][16];
    RowSum<TPR> sum{red};
    const int lane = TPR > 64 ? threadIdx.x : threadIdx.x & (TPR - 1);
    const int64_t row = (int64_t)blockIdx.x * NT + (TPR > 64 ? 0 : threadIdx.x / TPR);
    if (row >= a.rows) return;                         // whole teams; TPR > 64: the block has one team
    int n[NV];
    f8 x[NV], y[NV];
    typename Vec8<TX>::type rx[NV];
    typename Vec8<TY>::type ry[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + lane) * 8;
        n[j] = a.d - c;
        if (n[j] > 0) {
            rx[j] = load8_raw_n((const TX *)a.x + row * a.xs + c, n[j]);
            if (a.y) ry[j] = load8_raw_n((const TY *)a.y + row * a.ys + c, n[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        x[j] = n[j] > 0 ? widen<TX>(rx[j]) : splat8(0.f);
        y[j] = n[j] > 0 && a.y ? widen<TY>(ry[j]) : splat8(0.f);
    }
    if (a.y) {
        normalise<LN>(y, n, sum, a.eps, a.inv_d);
        const size_t g0 = (size_t)(row / a.rpg) * a.d;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * TPR + lane) * 8;
            if (n[j] <= 0) continue;
            f8 v = y[j];
            if (a.pw) v *= load8_either<TY>(a.pw, a.small32 & 2, c, n[j]);
            if (LN && a.pb) v += load8_either<TY>(a.pb, a.small32 & 2, c, n[j]);
            if (a.gate) v *= load8_either<TY>(a.gate, a.small32 & 1, g0 + c, n[j]);
            x[j] = x[j] * a.rs + v;
            store8_n((TX *)a.xn + row * a.d + c, x[j], n[j]);
        }
    }
    if (!a.pre) return;
    normalise<LN>(x, n, sum, a.eps, a.inv_d);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + lane) * 8;
        if (n[j] <= 0) continue;
        f8 v = x[j];
        if (a.qw) v *= load8_either<TY>(a.qw, a.small32 & 4, c, n[j]);
        if (LN && a.qb) v += load8_either<TY>(a.qb, a.small32 & 4, c, n[j]);
        store8_n((TY *)a.h + row * a.d + c, v, n[j]);
    }
}

// order of the partial sums: pre weight, post weight, pre bias, post bias (the biases for LayerNorm only)
template <class TX, class TY, int TPR, int NV, bool LN>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void block_norms_grad_kernel(const BnArgs a) {
    constexpr int NT = TPR <= 64 ? 256 / TPR : 1, NA = LN ? 4 : 2;
    __shared__ float red[2][16];
    __shared__ __attribute__((aligned(32))) float comb[NT > 1 ? 3 * TPR * 8 * NV : 1];
    RowSum<TPR> sum{red};
    const int lane = TPR > 64 ? threadIdx.x : threadIdx.x & (TPR - 1), team = TPR > 64 ? 0 : threadIdx.x / TPR;
    int n[NV];
    f8 acc[NA][NV], dg[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        n[j] = a.d - (j * TPR + lane) * 8;
#pragma unroll
        for (int k = 0; k < NA; ++k) acc[k][j] = splat8(0.f);
    }
    // A lane's share of the weights and of the gate row, fp32, in LDS that only it reads (no barriers): the row body uses them five
    // times, and every one of those would be a trip to L2.
    constexpr bool HELD = NV == 1;
    extern __shared__ __attribute__((aligned(16))) float held[];       // [3][2][threads][4]: post weight, pre weight, gate
    const int threads = blockDim.x;
    auto hold = [&](int k, const f8 &v) {
        *(float4 *)(held + (size_t)((2 * k) * threads + threadIdx.x) * 4) = float4{v[0], v[1], v[2], v[3]};
        *(float4 *)(held + (size_t)((2 * k + 1) * threads + threadIdx.x) * 4) = float4{v[4], v[5], v[6], v[7]};
    };
    auto held_at = [&](int k) {
        const float4 p = *(const float4 *)(held + (size_t)((2 * k) * threads + threadIdx.x) * 4), q = *(const float4 *)(held + (size_t)((2 * k + 1) * threads + threadIdx.x) * 4);
        return f8{p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
    };
    auto small = [&](const void *p, int bit, size_t at, int j, float none) {
        return p && n[j] > 0 ? load8_either<TY>(p, a.small32 & bit, at, n[j]) : splat8(none);
    };
    if constexpr (HELD) {
        hold(0, small(a.pw, 2, lane * 8, 0, 1.f));
        hold(1, small(a.qw, 4, lane * 8, 0, 1.f));
    }
    auto post_weight = [&](int j) { if constexpr (HELD) return held_at(0); else return small(a.pw, 2, (j * TPR + lane) * 8, j, 1.f); };
    auto pre_weight = [&](int j) { if constexpr (HELD) return held_at(1); else return small(a.qw, 4, (j * TPR + lane) * 8, j, 1.f); };
    auto gate_of = [&](int j, size_t g0) { if constexpr (HELD) return held_at(2); else return small(a.gate, 1, g0 + (j * TPR + lane) * 8, j, 1.f); };
    // Above 4096 columns a CU holds one workgroup: the next row is asked for as soon as this one's registers are free (8192 rows of bf16,
    // 5120 columns: 207 us without, 181 with; 8192 columns: 265 and 212).  Below, the registers that takes would cost a second
    // workgroup, which hides more; with fp32 rows and in the layer's form they would go to scratch.
    constexpr bool AHEAD = TPR == 1024 && NV == 1 && !LN && sizeof(TX) == 2;
    typename Vec8<TX>::type rx[NV], rgx[NV];
    typename Vec8<TY>::type ry_[NV], rgh[NV];
    auto fetch = [&](int64_t row) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * TPR + lane) * 8;
            if (n[j] > 0) {
                rx[j] = load8_raw_n((const TX *)a.x + row * a.xs + c, n[j]);
                if (a.y) ry_[j] = load8_raw_n((const TY *)a.y + row * a.ys + c, n[j]);
                if (a.gx) rgx[j] = load8_raw_n((const TX *)a.gx + row * a.gxs + c, n[j]);
                if (a.gh) rgh[j] = load8_raw_n((const TY *)a.gh + row * a.ghs + c, n[j]);
            }
        }
    };
    auto one_row = [&](int64_t row, size_t g0, int64_t next) __attribute__((always_inline)) {      // as a call its sums would live in memory
        f8 x[NV], y[NV], gx[NV], gh[NV];
        if constexpr (!AHEAD) fetch(row);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            x[j] = n[j] > 0 ? widen<TX>(rx[j]) : splat8(0.f);
            y[j] = n[j] > 0 && a.y ? widen<TY>(ry_[j]) : splat8(0.f);
            gx[j] = n[j] > 0 && a.gx ? widen<TX>(rgx[j]) : splat8(0.f);
            gh[j] = n[j] > 0 && a.gh ? widen<TY>(rgh[j]) : splat8(0.f);
        }
        if constexpr (AHEAD) if (next >= 0) fetch(next);
        float ry = 0.f;
        if (a.y) {
            ry = normalise<LN>(y, n, sum, a.eps, a.inv_d);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * TPR + lane) * 8;
                f8 v = y[j] * post_weight(j);
                if (LN) v += small(a.pb, 2, c, j, 0.f);
                x[j] = x[j] * a.rs + v * gate_of(j, g0);
            }
        }
        if (a.pre) {
            const float r = normalise<LN>(x, n, sum, a.eps, a.inv_d);
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                acc[0][j] += gh[j] * x[j];
                if constexpr (LN) acc[2][j] += gh[j];
                gh[j] *= pre_weight(j);
                s1 += sum8(gh[j] * x[j]);
                if (LN) s2 += sum8(gh[j]);
            }
            s1 = sum(s1) * a.inv_d;
            if (LN) s2 = sum(s2) * a.inv_d;
#pragma unroll
            for (int j = 0; j < NV; ++j) gx[j] += (gh[j] - s2 - x[j] * s1) * r;
        }
        const float back = a.y ? a.rs : 1.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (n[j] > 0) store8_n((TX *)a.dx + row * a.d + (j * TPR + lane) * 8, gx[j] * back, n[j]);
        if (!a.y) return;
        float t1 = 0.f, t2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * TPR + lane) * 8;
            const f8 w = post_weight(j);
            f8 v = y[j] * w;
            if (LN) v += small(a.pb, 2, c, j, 0.f);
            dg[j] += gx[j] * v;
            gx[j] *= gate_of(j, g0);
            if (n[j] < 8)                              // columns past d carry the LayerNorm means of gx: nothing of them is summed
#pragma unroll
                for (int e = 0; e < 8; ++e) if (e >= n[j]) gx[j][e] = 0.f;
            acc[1][j] += gx[j] * y[j];
            if constexpr (LN) acc[3][j] += gx[j];
            gx[j] *= w;
            t1 += sum8(gx[j] * y[j]);
            if (LN) t2 += sum8(gx[j]);
        }
        t1 = sum(t1) * a.inv_d;
        if (LN) t2 = sum(t2) * a.inv_d;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (n[j] > 0) store8_n((TY *)a.dy + row * a.d + (j * TPR + lane) * 8, (gx[j] - t2 - y[j] * t1) * ry, n[j]);
    };
    // adds the teams' registers: within a wave by lane distance, then the block's waves in order; the sum is valid in team 0
    auto join_teams = [&](f8 (&v)[NV]) {
        if constexpr (NT > 1) {
#pragma unroll
            for (int o = TPR; o < 64; o <<= 1)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[j][e] += __shfl_xor(v[j][e], o, 64);
            const int wave = threadIdx.x >> 6;
            __syncthreads();
            if (wave > 0 && (threadIdx.x & 63) < TPR)
#pragma unroll
                for (int j = 0; j < NV; ++j) *(f8 *)(comb + (size_t)((j * 3 + wave - 1) * TPR + lane) * 8) = v[j];
            __syncthreads();
            if (team == 0)
                for (int w = 0; w < 3; ++w)
#pragma unroll
                    for (int j = 0; j < NV; ++j) v[j] += *(const f8 *)(comb + (size_t)((j * 3 + w) * TPR + lane) * 8);
        }
    };
    auto clear = [&]() {
#pragma unroll
        for (int j = 0; j < NV; ++j) dg[j] = splat8(0.f);
    };
    auto put_gate = [&](int64_t g, int s) {
        if (!a.dgate) return;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * TPR + lane) * 8;
            if (n[j] <= 0) continue;
            if (a.S == 1) store8_either<TY>(a.dgate, a.small32 & 1, (size_t)g * a.d + c, dg[j], n[j]);
            else store8_n(a.gpart + ((size_t)g * a.S + s) * a.d + c, dg[j], n[j]);
        }
    };
    // Short runs of rows per gate (fewer than the block has teams): `a.cell` teams of one wave take a run.  Otherwise the block takes
    // `split_rows` rows of one gate row at a time.
    const bool few = NT > 1 && a.rpg < NT;
    const int cells = few ? NT / a.cell : 1, sub = few ? team & (a.cell - 1) : team;
    const int64_t items = few ? (a.G + cells - 1) / cells : a.G * a.S;
    for (int64_t w = blockIdx.x; w < items; w += gridDim.x) {
        const int64_t g = few ? w * cells + team / a.cell : w / a.S;
        const int s = few ? 0 : (int)(w - g * a.S);
        const int64_t end = (g + 1) * a.rpg, r0 = g * a.rpg + s * a.split_rows, r1 = few || r0 + a.split_rows > end ? end : r0 + a.split_rows;
        clear();
        if constexpr (HELD) if (g < a.G) hold(2, small(a.gate, 1, (size_t)g * a.d + lane * 8, 0, 1.f));
        if (g < a.G) {
            const int64_t step = few ? a.cell : NT;
            if constexpr (AHEAD) if (r0 + sub < r1) fetch(r0 + sub);
            for (int64_t r = r0 + sub; r < r1; r += step) one_row(r, (size_t)g * a.d, r + step < r1 ? r + step : -1);
        }
        if (!a.dgate) continue;
        if (few) {
            for (int o = TPR; o < a.cell * TPR; o <<= 1)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) dg[j][e] += __shfl_xor(dg[j][e], o, 64);
        } else join_teams(dg);
        if (sub == 0 && g < a.G) put_gate(g, s);
    }
    if (!a.part) return;
#pragma unroll
    for (int k = 0; k < NA; ++k) {
        join_teams(acc[k]);
        if (team == 0)
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (n[j] > 0) store8_n(a.part + ((size_t)blockIdx.x * NA + k) * a.d + (j * TPR + lane) * 8, acc[k][j], n[j]);
    }
}

// sums over the blocks' (weights) or a gate row's pieces: sixteen waves add a contiguous share each, then in wave order
struct BnJoin {
    const float *part, *gpart;
    void *out[4];
    void *dgate;
    int na, nblk, S, d, small32;
};
template <class TY> __device__ __forceinline__ void put1(void *p, bool f32, size_t at, float v) {
    if (f32) ((float *)p)[at] = v;
    else ((TY *)p)[at] = (TY)v;
}
template <class TY>
__global__ __launch_bounds__(1024) void block_norms_join_kernel(const BnJoin a) {
    __shared__ float q[16][64];
    const int col = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + col;
    const bool weight = (int)blockIdx.y < a.na;
    const int g = (int)blockIdx.y - a.na;
    if (weight && !a.out[blockIdx.y]) return;
    const int count = weight ? a.nblk : a.S;
    const float *src = weight ? a.part + (size_t)blockIdx.y * a.d : a.gpart + (size_t)g * a.S * a.d;
    const size_t step = weight ? (size_t)a.na * a.d : (size_t)a.d;
    const int per = (count + 15) / 16, k0 = w * per, k1 = k0 + per < count ? k0 + per : count;
    float s = 0.f;
    if (c < a.d) s = sum_strided(src + c, k0, k1, step);
    q[w][col] = s;
    __syncthreads();
    if (w != 0 || c >= a.d) return;
    s = q[0][col];
#pragma unroll
    for (int k = 1; k < 16; ++k) s += q[k][col];
    if (weight) put1<TY>(a.out[blockIdx.y], a.small32 & ((blockIdx.y & 1) ? 2 : 4), c, s);
    else put1<TY>(a.dgate, a.small32 & 1, (size_t)g * a.d + c, s);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
namespace {
constexpr int BN_MAX_D = 16384;
int lanes_for(int64_t d) {                             // lanes of a team: eight columns each
    const int64_t v = ceil_div(d, 8);
    return v <= 8 ? 8 : v <= 16 ? 16 : v <= 32 ? 32 : pow2_at_least(v, 64, 1024);
}
struct BnPlan {
    int tpr, nt, nblk, S, na, cell;
    int64_t split;
    size_t gpart, bytes;
};
BnPlan grad_plan(const dnag_block_norms_args &p) {
    BnPlan q;
    q.tpr = lanes_for(p.dim);
    q.nt = q.tpr <= 64 ? 256 / q.tpr : 1;
    q.na = p.layer_norm ? 4 : 2;
    const int64_t G = p.gate_rows, rpg = p.rows / G;
    // as many blocks as the chip holds at a time, or twice that: fewer partial sums than with a block per row.  Half of them, these and
    // twice as many, us, bf16: 65536 x 64 26, 22, 27; 65536 x 256 75, 49, 55; 32768 x 512 80, 52, 58; 16384 x 1024 101, 61, 53; 16384 x 2048
    // 128, 96, 102; 16384 x 4096 289, 197, 199; 8192 x 8192 378, 211, 224; 2048 x 16384 565, 345, 380; 1024 x 4096 29, 26, 34
    const int64_t target = q.tpr <= 64 || q.tpr == 512 ? 512 : q.tpr > 512 ? 256 : 1024;
    q.S = 1;
    if (rpg >= q.nt) {
        int64_t s = ceil_div(target, G), most = ceil_div(rpg, q.nt);
        if (s > most) s = most;
        q.split = ceil_div(rpg, s);
        q.S = (int)ceil_div(rpg, q.split);
    } else q.split = rpg;
    // a run of rows shared by as many teams of a wave as it has rows: one team for a run left the chip half empty (4096 runs of
    // 8 rows of 64 in fp32, LayerNorm: 36 us; shared by 8 teams: 20)
    q.cell = 1;
    while (q.cell * 2 <= rpg && q.cell * 2 * q.tpr <= 64) q.cell *= 2;
    const int64_t items = rpg >= q.nt ? G * q.S : ceil_div(G, q.nt / q.cell);
    q.nblk = (int)(items < target ? items : target);
    q.gpart = align256((size_t)q.nblk * q.na * p.dim * 4);
    q.bytes = q.gpart + (q.S > 1 ? (size_t)G * q.S * p.dim * 4 : 0);
    return q;
}
int check(const dnag_block_norms_args *p) {
    if (!p) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    if (!dtype_known(p->dtype)) return dnag_fail(DNAG_E_ARG, "unknown dtype %d", p->dtype);
    if (p->x_dtype != p->dtype && p->x_dtype != DNAG_F32) return dnag_fail(DNAG_E_ARG, "the residual stream has dtype %d: the branch's (%d) or fp32 are built", p->x_dtype, p->dtype);
    if (p->dim < 1 || p->dim > BN_MAX_D) return dnag_fail(DNAG_E_ARG, "dim=%lld out of range (1 .. %d)", (long long)p->dim, BN_MAX_D);
    if (p->rows < 0 || p->rows > 0x7fffffffll) return dnag_fail(DNAG_E_ARG, "rows=%lld out of range", (long long)p->rows);
    if (p->gate_rows < 1 || (p->rows > 0 && p->rows % p->gate_rows)) return dnag_fail(DNAG_E_ARG, "%lld rows do not divide into %lld gate rows", (long long)p->rows, (long long)p->gate_rows);
    if (!p->layer_norm && (p->post_bias || p->pre_bias)) return dnag_fail(DNAG_E_ARG, "RMSNorm has no bias");
    if (!p->y && !p->pre) return dnag_fail(DNAG_E_ARG, "without y there is only the norm in front: pre must be set");
    if (!p->y && (p->gate || p->post_weight || p->post_bias)) return dnag_fail(DNAG_E_ARG, "gate and post norm need y");
    if (!p->pre && (p->pre_weight || p->pre_bias)) return dnag_fail(DNAG_E_ARG, "pre_weight / pre_bias without pre");
    if (p->x_stride < p->dim || (p->y && p->y_stride < p->dim)) return dnag_fail(DNAG_E_ARG, "a row stride is smaller than dim");
    return 0;
}
BnArgs common_args(const dnag_block_norms_args &p) {
    BnArgs a = {};
    a.x = p.x; a.y = p.y; a.gate = p.gate; a.pw = p.post_weight; a.pb = p.post_bias; a.qw = p.pre_weight; a.qb = p.pre_bias;
    a.xs = p.x_stride; a.ys = p.y_stride;
    a.rows = p.rows; a.G = p.gate_rows; a.rpg = p.rows / p.gate_rows;
    a.d = (int)p.dim; a.pre = p.pre; a.small32 = p.small_f32;
    a.rs = p.residual_scale; a.eps = p.eps; a.inv_d = 1.0f / (float)p.dim;
    return a;
}
template <class TX, class TY, int TPR, int NV, bool LN>
int launch(const BnArgs &a, bool grad, unsigned blocks, hipStream_t st) {
    // a team above 64 lanes is the workgroup: whole waves, as many as the row needs (4100 columns: 9, not 16)
    const int threads = TPR <= 64 ? 256 : NV > 1 ? TPR : (int)(ceil_div(a.d, 512) * 64);
    if (int rc = grid_fits(blocks, threads)) return rc;
    if (grad) {
        const size_t lds = NV == 1 ? (size_t)3 * threads * 32 : 0;
        static LdsLimit limit;
        TOK_TRY(limit.allow((const void *)block_norms_grad_kernel<TX, TY, TPR, NV, LN>, lds));
        hipLaunchKernelGGL((block_norms_grad_kernel<TX, TY, TPR, NV, LN>), dim3(blocks), dim3(threads), lds, st, a);
    } else hipLaunchKernelGGL((block_norms_kernel<TX, TY, TPR, NV, LN>), dim3(blocks), dim3(threads), 0, st, a);
    return 0;
}
template <class TX, class TY, bool LN>
int launch_width(const BnArgs &a, int tpr, bool grad, unsigned blocks, hipStream_t st) {
    switch (tpr) {
        case 8: return launch<TX, TY, 8, 1, LN>(a, grad, blocks, st);
        case 16: return launch<TX, TY, 16, 1, LN>(a, grad, blocks, st);
        case 32: return launch<TX, TY, 32, 1, LN>(a, grad, blocks, st);
        case 64: return launch<TX, TY, 64, 1, LN>(a, grad, blocks, st);
        case 128: return launch<TX, TY, 128, 1, LN>(a, grad, blocks, st);
        case 256: return launch<TX, TY, 256, 1, LN>(a, grad, blocks, st);
        case 512: return launch<TX, TY, 512, 1, LN>(a, grad, blocks, st);
        default:
            if (a.d <= 8192) return launch<TX, TY, 1024, 1, LN>(a, grad, blocks, st);
            return launch<TX, TY, 1024, 2, LN>(a, grad, blocks, st);
    }
}
template <class TX, class TY>
int launch_types(const dnag_block_norms_args &p, const BnArgs &a, int tpr, bool grad, unsigned blocks) {
    hipStream_t st = (hipStream_t)p.stream;
    if (int rc = p.layer_norm ? launch_width<TX, TY, true>(a, tpr, grad, blocks, st) : launch_width<TX, TY, false>(a, tpr, grad, blocks, st)) return rc;
    TOK_TRY(hipGetLastError());
    return 0;
}
int launch_all(const dnag_block_norms_args &p, const BnArgs &a, int tpr, bool grad, unsigned blocks) {
    if (p.dtype == DNAG_F32) return launch_types<float, float>(p, a, tpr, grad, blocks);
    if (p.dtype == DNAG_BF16) return p.x_dtype == DNAG_F32 ? launch_types<float, tbf16>(p, a, tpr, grad, blocks) : launch_types<tbf16, tbf16>(p, a, tpr, grad, blocks);
    return p.x_dtype == DNAG_F32 ? launch_types<float, tf16>(p, a, tpr, grad, blocks) : launch_types<tf16, tf16>(p, a, tpr, grad, blocks);
}
}  // namespace

extern "C" size_t dnag_block_norms_args_bytes(void) { return sizeof(dnag_block_norms_args); }

extern "C" int dnag_block_norms_forward(const dnag_block_norms_args *p) {
    if (int rc = check(p)) return rc;
    if (p->rows == 0) return 0;
    if (!p->x || (p->y && !p->x_new) || (p->pre && !p->h)) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    BnArgs a = common_args(*p);
    a.xn = p->x_new; a.h = p->h;
    const int tpr = lanes_for(p->dim);
    return launch_all(*p, a, tpr, false, (unsigned)ceil_div(p->rows, tpr <= 64 ? 256 / tpr : 1));
}

extern "C" size_t dnag_block_norms_grad_workspace_bytes(const dnag_block_norms_args *p) {
    if (check(p) || p->rows == 0) return 0;
    return grad_plan(*p).bytes;
}

extern "C" int dnag_block_norms_grad(const dnag_block_norms_args *p) {
    if (int rc = check(p)) return rc;
    if (p->rows == 0) return dnag_fail(DNAG_E_ARG, "no rows: the gradients of the weights are zeros, nothing is launched");
    if (!p->x || !p->dx || (p->y && !p->dy)) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    if ((p->d_gate && !p->gate) || (p->d_post_weight && !p->post_weight) || (p->d_post_bias && !p->post_bias) || (p->d_pre_weight && !p->pre_weight) ||
        (p->d_pre_bias && !p->pre_bias)) return dnag_fail(DNAG_E_ARG, "a gradient is asked for an input that is not there");
    if ((p->grad_x && p->grad_x_stride < p->dim) || (p->grad_h && p->grad_h_stride < p->dim)) return dnag_fail(DNAG_E_ARG, "a row stride is smaller than dim");
    if (p->grad_h && !p->pre) return dnag_fail(DNAG_E_ARG, "grad_h without pre");
    const BnPlan q = grad_plan(*p);
    if (!p->workspace || p->workspace_bytes < q.bytes) return dnag_fail(DNAG_E_WORKSPACE, "workspace has %zu bytes, %zu are needed", p->workspace_bytes, q.bytes);
    BnArgs a = common_args(*p);
    a.gx = p->grad_x; a.gh = p->grad_h; a.gxs = p->grad_x_stride; a.ghs = p->grad_h_stride;
    a.dx = p->dx; a.dy = p->dy; a.dgate = p->d_gate;
    a.S = q.S; a.split_rows = q.split; a.cell = q.cell;
    const bool weights = p->d_post_weight || p->d_post_bias || p->d_pre_weight || p->d_pre_bias;
    a.part = weights ? (float *)p->workspace : nullptr;
    a.gpart = (float *)((char *)p->workspace + q.gpart);
    if (int rc = launch_all(*p, a, q.tpr, true, (unsigned)q.nblk)) return rc;
    const bool gates = p->d_gate && q.S > 1;
    if (!weights && !gates) return 0;
    BnJoin j = {};
    j.part = a.part; j.gpart = a.gpart;
    j.out[0] = p->d_pre_weight; j.out[1] = p->d_post_weight; j.out[2] = p->d_pre_bias; j.out[3] = p->d_post_bias;
    j.dgate = p->d_gate;
    j.na = weights ? q.na : 0; j.nblk = q.nblk; j.S = q.S; j.d = (int)p->dim; j.small32 = p->small_f32;
    // (without weights the part's arrays are not there: the grid's second axis holds the gate rows only)
    const dim3 grid((unsigned)ceil_div(p->dim, 64), (unsigned)(j.na + (gates ? p->gate_rows : 0)));
    hipStream_t st = (hipStream_t)p->stream;
    if (p->dtype == DNAG_F32) hipLaunchKernelGGL((block_norms_join_kernel<float>), grid, dim3(1024), 0, st, j);
    else if (p->dtype == DNAG_BF16) hipLaunchKernelGGL((block_norms_join_kernel<tbf16>), grid, dim3(1024), 0, st, j);
    else hipLaunchKernelGGL((block_norms_join_kernel<tf16>), grid, dim3(1024), 0, st, j);
    TOK_TRY(hipGetLastError());
    return 0;
}
