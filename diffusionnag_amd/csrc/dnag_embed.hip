// Embedding lookup with scaling and its gradient.
//   forward:   out[t] = scale * W[ids[t]], a row of zeros for an id outside 0 .. V - 1
//   gradient:  dW[v] = scale * sum over t with ids[t] = v of dout[t], in the order of t, in fp32, rounded once
// Both are bound by HBM: the forward reads T rows and writes T, the gradient reads T rows and writes V.
//
// The gradient sums rows by token without atomics, so that it gives the same bits every time.
//   V <= EMB_FEW (the architecture vocabularies): every team of lanes keeps a table [V][64 columns] of its own in LDS and walks
//     its rows in order; tables are added in team order, blocks' tables in block order (second launch).
//   otherwise: the positions are sorted by (token, position) -- in LDS by one workgroup up to EMB_SORT_LDS rows, by a stable
//     least-significant-digit radix sort above --, teams walk chunks of the sorted list and write a token's row when it lies
//     inside the chunk; the pieces of tokens that cross chunk borders go to a workspace, and the last launch adds them in
//     chunk order and writes the zero rows of the tokens that do not occur.
#include "dnag_token_common.h"

// Tokens whose rows of 64 columns are kept for each of 32 teams: 8 KB of LDS a token, 128 KB at 16.  In us, this and the sorted list, 32768
// rows: 12 x 64 fp32 8 and 23, 16 x 64 9 and 23, 9 x 1024 bf16 23 and 36, 16 x 1024 38 and 36; with room for 18 (144 KB), 18 x 64 9 and 22,
// 18 x 1024 40 and 35: wide rows are better sorted from 16 on, narrow ones not before the LDS ends.
#define EMB_FEW 16
// Rows that one workgroup sorts in LDS, three launches in all instead of four to eight: its time grows with the rows, the radix sort's with the
// passes over the tokens' digits.  In us, this and the radix sort, bf16: 1024 rows over 100 x 64 24 and 18, 300 x 512 23 and 26, 32000 x 512
// 34 and 44, 100000 x 64 54 and 85; 2048 rows 30 and 18, 29 and 27, 41 and 43, 60 and 80; 4096 rows 46 and 19, 46 and 29, 59 and 43,
// 77 and 78.
#define EMB_SORT_LDS 2048

template <class I> __device__ __forceinline__ uint32_t emb_key(const I *ids, size_t t, int64_t V, int64_t pad) {
    const int64_t v = (int64_t)ids[t];
    return v >= 0 && v < V && v != pad ? (uint32_t)v : (uint32_t)V;
}

// ---- forward: TPR lanes per row, eight columns per lane and step -----------------------------------------------------
template <class T, class I>
__global__ __launch_bounds__(256) void embed_forward_kernel(const I *__restrict__ ids, int64_t rows, const T *__restrict__ w, int64_t wstride,
                                                            int64_t V, int d, float scale, T *__restrict__ out, int tpr) {
    const int lane = threadIdx.x & (tpr - 1), per = 256 / tpr;
    const int64_t t = (int64_t)blockIdx.x * per + threadIdx.x / tpr;
    if (t >= rows) return;
    const int64_t v = (int64_t)ids[t];
    const bool real = v >= 0 && v < V;
    const T *src = w + (real ? v : 0) * wstride;
    T *dst = out + t * d;
    for (int c = (blockIdx.y * tpr + lane) * 8; c < d; c += gridDim.y * tpr * 8) {
        const int n = d - c < 8 ? d - c : 8;
        f8 x = splat8(0.f);
        if (real) x = load8_n(src + c, n) * scale;
        store8_n(dst + c, x, n);
    }
}

// ---- gradient, few tokens --------------------------------------------------------------------------------------------
// blockIdx.y: tile of 64 columns, eight lanes of eight columns; 32 teams, each with rows first + team * len ...
template <class T, class I>
__global__ __launch_bounds__(256) void embed_few_kernel(const I *__restrict__ ids, int64_t rows, const T *__restrict__ grad, int64_t gstride,
                                                        int V, int64_t pad, int d, float scale, int64_t rows_per_block,
                                                        float *__restrict__ part, T *__restrict__ out) {
    extern __shared__ float tab[];                     // [32][V][64]
    const int lane = threadIdx.x & 7, team = threadIdx.x >> 3;
    const int c = blockIdx.y * 64 + lane * 8;
    const int n = d - c < 8 ? d - c : 8;
    float *mine = tab + (size_t)team * V * 64 + lane * 8;
    for (int v = 0; v < V; ++v) *(f8 *)(mine + v * 64) = splat8(0.f);
    const int64_t b0 = (int64_t)blockIdx.x * rows_per_block, b1 = b0 + rows_per_block < rows ? b0 + rows_per_block : rows;
    const int64_t len = (b1 - b0 + 31) / 32, t0 = b0 + team * len, t1 = t0 + len < b1 ? t0 + len : b1;
    if (n > 0)
        for (int64_t t = t0; t < t1; t += 4) {
            typename Vec8<T>::type x[4];
            uint32_t k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t tt = t + u < t1 ? t + u : t1 - 1;
                k[u] = t + u < t1 ? emb_key(ids, tt, V, pad) : (uint32_t)V;
                x[u] = load8_raw_n(grad + tt * gstride + c, n);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k[u] < (uint32_t)V) *(f8 *)(mine + k[u] * 64) += widen<T>(x[u]);
        }
    __syncthreads();
    for (int i = threadIdx.x; i < V * 64; i += 256) {
        const int v = i >> 6, cc = blockIdx.y * 64 + (i & 63);
        if (cc >= d) continue;
        float s = 0.f;
        for (int q = 0; q < 32; ++q) s += tab[(size_t)q * V * 64 + i];
        if (part) part[((size_t)blockIdx.x * V + v) * d + cc] = s;
        else out[(size_t)v * d + cc] = (T)(s * scale);
    }
}
// out[i] = scale * sum of nblk tables: sixteen waves add a contiguous share of the blocks each, then in wave order
template <class T>
__global__ __launch_bounds__(1024) void embed_few_join_kernel(const float *__restrict__ part, int nblk, int64_t n, float scale, T *__restrict__ out) {
    __shared__ float q[16][64];
    const int col = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t i = (int64_t)blockIdx.x * 64 + col;
    const int per = (nblk + 15) / 16, a = w * per, b = a + per < nblk ? a + per : nblk;
    float s = 0.f;
    if (i < n) s = sum_strided(part + i, a, b, (size_t)n);
    q[w][col] = s;
    __syncthreads();
    if (w == 0 && i < n) {
        s = q[0][col];
#pragma unroll
        for (int k = 1; k < 16; ++k) s += q[k][col];
        out[i] = (T)(s * scale);
    }
}

// ---- gradient, sort --------------------------------------------------------------------------------------------------
// block 0: all pairs in LDS, bitonic (the pairs are distinct, so the order is the stable one); other blocks: last[] = 0
template <class I>
__global__ __launch_bounds__(1024) void embed_sort_lds_kernel(const I *__restrict__ ids, int rows, int n2, int64_t V, int64_t pad,
                                                              uint32_t *__restrict__ key, uint32_t *__restrict__ pos, uint32_t *__restrict__ last) {
    extern __shared__ uint64_t pr[];
    if (blockIdx.x > 0) {
        for (int64_t v = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; v < V; v += (int64_t)(gridDim.x - 1) * 1024) last[v] = 0;
        return;
    }
    for (int i = threadIdx.x; i < n2; i += 1024) pr[i] = i < rows ? ((uint64_t)emb_key(ids, i, V, pad) << 32) | (uint32_t)i : ~0ull;
    for (int k = 2; k <= n2; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (int p = threadIdx.x; p < n2 / 2; p += 1024) {
                const int i = 2 * p - (p & (j - 1));              // the p-th index whose bit j is clear
                const uint64_t a = pr[i], b = pr[i + j];
                if ((a > b) == ((i & k) == 0)) { pr[i] = b; pr[i + j] = a; }
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < rows; i += 1024) { key[i] = (uint32_t)(pr[i] >> 32); pos[i] = (uint32_t)pr[i]; }
}

// Rows of tokens that do not occur, written by workgroups that ride along with the sort's launches (those keep 32 of 256 CUs
// busy): tokens [v0, v1) whose `last` is 0, `units` 16-bit words each.
struct EmbFill {
    const uint32_t *last;
    uint16_t *out;
    int64_t v0, v1, units;
    int first;                         // workgroups of the sort itself
};
__device__ __forceinline__ void emb_fill(const EmbFill &f) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    const u16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    const int64_t wgs = gridDim.x - f.first;
    for (int64_t b = f.v0 + (blockIdx.x - f.first); b < f.v1; b += 64 * wgs) {       // 64 tokens at a time, a lane asks for each
        const int64_t mine = b + (threadIdx.x & 63) * wgs;
        uint64_t empty = __ballot(mine < f.v1 && f.last[mine < f.v1 ? mine : b] == 0);       // the same in every wave
        for (; empty; empty &= empty - 1) {
            uint16_t *dst = f.out + (b + (__ffsll((long long)empty) - 1) * wgs) * f.units;
            for (int64_t c = threadIdx.x * 8; c < f.units; c += blockDim.x * 8) {
                if (f.units - c >= 8) __builtin_memcpy(dst + c, &zero, 16);
                else
                    for (int64_t e = c; e < f.units; ++e) dst[e] = 0;
            }
        }
    }
}

// Stable radix sort, digits of eight bits.  A block owns a contiguous range of the list and each of its four waves a
// contiguous quarter; at most EMB_MAXB blocks, so that every block sums the others' histograms by itself (no scan launch).
// With 64, 128 and 256 of them, us for the whole gradient over 32000 x 64 bf16: 131072 rows 60, 58, 58; 270000 rows 98, 86, 85; 1000000 rows 222,
// 164, 139.  Up to 131072 rows a block has at least 1024 and the number makes no difference.
#define EMB_MAXB 128
template <class I>
__device__ __forceinline__ uint32_t emb_pass_key(const I *ids, const uint32_t *kin, int64_t i, int64_t V, int64_t pad) {
    return ids ? emb_key(ids, i, V, pad) : kin[i];
}
template <class I>
__global__ __launch_bounds__(256) void embed_hist_kernel(const I *__restrict__ ids, const uint32_t *__restrict__ kin, int64_t rows, int64_t per_block,
                                                         int64_t V, int64_t pad, int shift, uint32_t *__restrict__ hist, uint32_t *__restrict__ last, EmbFill fill) {
    if ((int)blockIdx.x >= fill.first) { emb_fill(fill); return; }
    __shared__ uint32_t h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b0 = blockIdx.x * per_block, b1 = b0 + per_block < rows ? b0 + per_block : rows;
    for (int64_t i = b0 + threadIdx.x; i < b1; i += 256) atomicAdd(&h[(emb_pass_key(ids, kin, i, V, pad) >> shift) & 255], 1u);   // counts: any order
    if (last)
        for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < V; v += (int64_t)fill.first * 256) last[v] = 0;
    __syncthreads();
    hist[blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}
template <class I>
__global__ __launch_bounds__(256) void embed_scatter_kernel(const I *__restrict__ ids, const uint32_t *__restrict__ kin, const uint32_t *__restrict__ pin,
                                                            int64_t rows, int64_t per_block, int64_t V, int64_t pad, int shift,
                                                            const uint32_t *__restrict__ hist, uint32_t *__restrict__ kout, uint32_t *__restrict__ pout,
                                                            uint32_t *__restrict__ mark, EmbFill fill) {
    if ((int)blockIdx.x >= fill.first) { emb_fill(fill); return; }
    __shared__ uint32_t cnt[4][256], scan[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // base of digit tid for this block: digits before it in the whole list, then the same digit in earlier blocks
    uint32_t total = 0, before = 0;
#pragma unroll 8
    for (int b = 0; b < fill.first; ++b) {
        const uint32_t x = hist[b * 256 + tid];
        total += x;
        before += b < (int)blockIdx.x ? x : 0;
    }
    scan[tid] = total;
#pragma unroll
    for (int w = 0; w < 4; ++w) cnt[w][tid] = 0;
    __syncthreads();
    for (int o = 1; o < 256; o *= 2) {
        const uint32_t x = tid >= o ? scan[tid - o] : 0;
        __syncthreads();
        scan[tid] += x;
        __syncthreads();
    }
    const uint32_t base = scan[tid] - total + before;
    const int64_t b0 = blockIdx.x * per_block, b1 = b0 + per_block < rows ? b0 + per_block : rows;
    const int64_t quarter = (per_block / 4 + 63) / 64 * 64;
    const int64_t w0 = b0 + wave * quarter < b1 ? b0 + wave * quarter : b1, w1 = wave < 3 && w0 + quarter < b1 ? w0 + quarter : b1;
    for (int64_t i = w0 + lane; i < w1; i += 64) atomicAdd(&cnt[wave][(emb_pass_key(ids, kin, i, V, pad) >> shift) & 255], 1u);
    __syncthreads();
    uint32_t at = base;
#pragma unroll
    for (int w = 0; w < 4; ++w) { const uint32_t x = cnt[w][tid]; cnt[w][tid] = at; at += x; }
    __syncthreads();
    for (int64_t i0 = w0; i0 < w1; i0 += 64) {          // 64 positions at a time, in order
        const int64_t i = i0 + lane;
        const bool on = i < w1;
        const uint32_t k = on ? emb_pass_key(ids, kin, i, V, pad) : 0u, dig = (k >> shift) & 255;
        uint64_t same = __ballot(on);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint64_t m = __ballot((dig >> b) & 1);
            same &= (dig >> b) & 1 ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        uint32_t first = 0;
        if (on) first = cnt[wave][dig];
        wave_fence();
        if (on) {
            kout[first + rank] = k;
            pout[first + rank] = pin ? pin[i] : (uint32_t)i;
            if (mark && k < (uint32_t)V) mark[k] = ~0u;          // the token occurs (any order, one value)
            if (rank == 0) cnt[wave][dig] = first + (uint32_t)__popcll(same);
        }
        wave_fence();
    }
}

// Sums over the sorted list: a team of TPR lanes (TPR * 8 columns) walks `chunk` (8 to 64) entries.  The lanes fetch TPR of the
// entries at once, one each, so that the rows' addresses are known before the first row is asked for; eight rows are
// under way at a time (fetching four entries, then their rows, in turn: 94 us for 32768 x 2048 bf16; this: 58, 2.3 TB/s of the
// gradient's rows).
template <class T, int TPR>
__global__ __launch_bounds__(256) void embed_sum_kernel(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, int64_t rows,
                                                        const T *__restrict__ grad, int64_t gstride, uint32_t V, int d, float scale, int chunk, int ntile,
                                                        T *__restrict__ out, uint32_t *__restrict__ last, float *__restrict__ part) {
    typedef typename Vec8<T>::type raw8;
    const int lane = threadIdx.x & (TPR - 1);
    const int in_block = TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / TPR;
    const int64_t unit = (int64_t)blockIdx.x * (256 / TPR) + in_block;
    const int64_t ch = unit / ntile;
    const int tile = (int)(unit - ch * ntile);
    const int64_t i0 = ch * chunk, i1 = i0 + chunk < rows ? i0 + chunk : rows;
    if (i0 >= rows) return;                            // whole teams
    const int c = (tile * TPR + lane) * 8, n = d - c < 8 ? d - c : 8;
    f8 acc = splat8(0.f);
    uint32_t cur = TPR == 64 ? __builtin_amdgcn_readfirstlane(key[i0]) : key[i0];
    bool older = i0 > 0 && key[i0 - 1] == cur;          // the token's rows began in an earlier chunk
    const uint32_t next = i1 < rows ? key[i1] : ~0u;
    auto flush = [&](int64_t end, bool more) {          // the rows of `cur` before `end`; more: they go on in the next chunk
        if (tile == 0 && lane == 0 && !more) last[cur] = (uint32_t)end;
        if (n <= 0) return;
        if (!older && !more) store8_n(out + (size_t)cur * d + c, acc * scale, n);
        else store8_n(part + ((size_t)ch * 2 + (older ? 0 : 1)) * d + c, acc, n);
    };
    for (int64_t b = i0; b < i1; b += TPR) {            // entries b .. b + TPR - 1, one per lane
        const int64_t mine = b + lane < i1 ? b + lane : i1 - 1;
        const uint32_t kk = key[mine], pp = pos[mine];
        const int m = (int)(i1 - b < TPR ? i1 - b : TPR);
        for (int g = 0; g < m; g += 8) {
            uint32_t k[8];
            raw8 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int src = g + u < m ? g + u : m - 1;
                // one team is the wave: scalar registers and branches
                const uint32_t kv = TPR == 64 ? __builtin_amdgcn_readlane(kk, src) : __shfl(kk, src, TPR);
                const uint32_t pv = TPR == 64 ? __builtin_amdgcn_readlane(pp, src) : __shfl(pp, src, TPR);
                k[u] = g + u < m ? kv : cur;
                const T *p = grad + (size_t)pv * gstride + c;
                x[u] = load8_raw_n(p, n);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (g + u < m) {
                    if (k[u] != cur) {
                        if (cur < V) flush(b + g + u, false);
                        acc = splat8(0.f);
                        cur = k[u];
                        older = false;
                    }
                    acc += widen<T>(x[u]);
                }
            if (cur >= V) return;                       // the dropped ones are the list's end
        }
    }
    if (cur < V) flush(i1, next == cur);
}

// Tokens whose rows cross chunk borders: their pieces in chunk order.  A workgroup for each chunk and 256 columns; the one whose chunk
// holds such a token's first row, but not its last, adds the token's pieces: sixteen shares of consecutive pieces, joined in
// order.  The workgroups behind them clear the rows of tokens that do not occur, where the sort has not done it.
template <class T>
__global__ __launch_bounds__(512) void embed_join_kernel(const uint32_t *__restrict__ key, const uint32_t *__restrict__ last, int64_t rows, uint32_t V,
                                                         const float *__restrict__ part, int chunk, int ntile, int d, float scale, T *__restrict__ out, EmbFill fill) {
    if ((int64_t)blockIdx.x >= fill.first) { emb_fill(fill); return; }
    __shared__ __attribute__((aligned(32))) float sh[512 * 8];
    const int64_t ch = blockIdx.x / ntile, i0 = ch * chunk, i1 = i0 + chunk;
    if (i1 >= rows) return;
    const uint32_t cur = key[i1 - 1], after = key[i1], prior = i0 > 0 ? key[i0 - 1] : ~0u;
    if (cur >= V || after != cur || prior == cur) return;
    const uint32_t count = (last[cur] - 1) / chunk - (uint32_t)ch + 1, each = (count + 15) / 16;
    const int cl = threadIdx.x & 31, share = threadIdx.x >> 5, c = ((int)(blockIdx.x - ch * ntile) * 32 + cl) * 8, n = d - c;
    const uint32_t a = share * each, b = a + each < count ? a + each : count;
    const float *src = part + (size_t)ch * 2 * d + c;  // piece 0 is the chunk's second one, the others are first ones
    f8 s = splat8(0.f);
    if (n >= 8)
        for (uint32_t k = a; k < b; k += 8) {           // eight at a time, the last ones too (a remainder would wait for each)
            f8 x[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) { const uint32_t q = k + u < b ? k + u : b - 1; x[u] = load8(src + ((size_t)q * 2 + (q == 0 ? 1 : 0)) * d); }
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) if (k + u < b) s += x[u];
        }
    else if (n > 0)
        for (uint32_t k = a; k < b; ++k) s += load8_n(src + ((size_t)k * 2 + (k == 0 ? 1 : 0)) * d, n);
    *(f8 *)(sh + threadIdx.x * 8) = s;
    __syncthreads();
    if (share != 0 || n <= 0) return;
    for (int q = 1; q < 16; ++q) s += *(const f8 *)(sh + (q * 32 + cl) * 8);
    store8_n(out + (size_t)cur * d + c, s * scale, n);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
namespace {
constexpr int64_t JOIN_CLEAR = 1024;   // workgroups behind the join's that clear rows, at most
struct GradPlan {
    bool few = false, lds = false;
    int64_t per_block = 0;             // few: rows per block; radix sort: list entries per block
    int nblk = 0, chunk = 0, nchunk = 0, passes = 0, jtile = 0;      // jtile: the join's tiles of 256 columns
    size_t part = 0, key[2] = {}, pos[2] = {}, hist = 0, last = 0, bytes = 0;      // offsets into the workspace
};

GradPlan grad_plan(int64_t rows, int64_t V, int64_t d) {
    GradPlan p;
    const int64_t tiles = ceil_div(d, 64);
    if (V <= EMB_FEW) {
        p.few = true;
        // enough blocks for the chip over rows and column tiles, at least four rows for a team
        int64_t nblk = ceil_div(512, tiles);
        p.per_block = ceil_div(rows, nblk);
        if (p.per_block < 128) p.per_block = 128;
        p.nblk = (int)(rows ? ceil_div(rows, p.per_block) : 1);
        p.bytes = p.nblk > 1 ? (size_t)p.nblk * V * d * 4 : 0;
        return p;
    }
    p.lds = rows <= EMB_SORT_LDS;
    const int64_t wide = ceil_div(d, 512);
    p.chunk = 64;                      // fewer pieces, but no fewer waves than eight for each of 256 CUs
    while (p.chunk > 8 && ceil_div(rows, p.chunk) * wide < 4096) p.chunk /= 2;
    p.nchunk = (int)ceil_div(rows, p.chunk);
    p.jtile = (int)ceil_div(d, 256);
    if (!p.lds) {
        p.per_block = ceil_div(ceil_div(rows, EMB_MAXB), 256) * 256;
        if (p.per_block < 1024) p.per_block = 1024;
        p.nblk = (int)ceil_div(rows, p.per_block);
        p.passes = 1;
        while (p.passes < 4 && (V >> (8 * p.passes)) > 0) ++p.passes;       // keys 0 .. V
    }
    size_t o = 0;
    auto take = [&](size_t n) { const size_t at = o; o += align256(n); return at; };
    for (int k = 0; k < (p.lds ? 1 : 2); ++k) { p.key[k] = take(rows * 4); p.pos[k] = take(rows * 4); }
    p.hist = take(p.lds ? 0 : EMB_MAXB * 256 * 4);
    p.last = take(V * 4);
    p.part = take((size_t)p.nchunk * 2 * d * 4);
    p.bytes = o;
    return p;
}

int check_embed(int64_t rows, int64_t V, int64_t d, int64_t stride, int dtype, int ids_bytes) {
    if (!dtype_known(dtype)) return dnag_fail(DNAG_E_ARG, "unknown dtype %d", dtype);
    if (ids_bytes != 4 && ids_bytes != 8) return dnag_fail(DNAG_E_ARG, "ids of %d bytes (4 or 8 are built)", ids_bytes);
    if (rows < 0 || rows > 0x7fffffffll) return dnag_fail(DNAG_E_ARG, "rows=%lld out of range", (long long)rows);
    if (V < 1 || V > 0x7ffffffell) return dnag_fail(DNAG_E_ARG, "num_tokens=%lld out of range", (long long)V);
    if (d < 1 || d > (1 << 20)) return dnag_fail(DNAG_E_ARG, "dim=%lld out of range (1 .. 2^20)", (long long)d);
    if (stride < d) return dnag_fail(DNAG_E_ARG, "row stride %lld is smaller than dim %lld", (long long)stride, (long long)d);
    return 0;
}

template <class T, class I>
int forward_t(const void *ids, int64_t rows, const void *w, int64_t ws, int64_t V, int64_t d, float scale, void *out, hipStream_t st) {
    const int tpr = pow2_at_least(ceil_div(d, 8), 1, 256);
    const int64_t bx = ceil_div(rows, 256 / tpr);
    if (int rc = grid_fits(bx, 256)) return rc;
    hipLaunchKernelGGL((embed_forward_kernel<T, I>), dim3((unsigned)bx, (unsigned)ceil_div(d, (int64_t)tpr * 8)), dim3(256), 0, st,
                       (const I *)ids, rows, (const T *)w, ws, V, (int)d, scale, (T *)out, tpr);
    TOK_TRY(hipGetLastError());
    return 0;
}

template <class T, class I>
int grad_t(const GradPlan &p, const void *ids, int64_t rows, const void *grad, int64_t gs, int64_t V, int64_t d, float scale, int64_t pad,
           void *out, char *ws, hipStream_t st) {
    const I *id = (const I *)ids;
    const T *g = (const T *)grad;
    if (p.few) {
        const size_t lds = (size_t)32 * V * 64 * 4;
        auto kern = embed_few_kernel<T, I>;
        static LdsLimit limit;
        TOK_TRY(limit.allow((const void *)kern, lds));
        float *part = p.nblk > 1 ? (float *)ws : nullptr;
        hipLaunchKernelGGL(kern, dim3(p.nblk, (unsigned)ceil_div(d, 64)), dim3(256), lds, st, id, rows, g, gs, (int)V, pad, (int)d, scale, p.per_block, part, (T *)out);
        TOK_TRY(hipGetLastError());
        if (part) {
            hipLaunchKernelGGL((embed_few_join_kernel<T>), dim3((unsigned)ceil_div(V * d, 64)), dim3(1024), 0, st, part, p.nblk, V * d, scale, (T *)out);
            TOK_TRY(hipGetLastError());
        }
        return 0;
    }
    uint32_t *key[2] = {(uint32_t *)(ws + p.key[0]), (uint32_t *)(ws + p.key[1])}, *pos[2] = {(uint32_t *)(ws + p.pos[0]), (uint32_t *)(ws + p.pos[1])};
    uint32_t *hist = (uint32_t *)(ws + p.hist), *last = (uint32_t *)(ws + p.last);
    float *part = (float *)(ws + p.part);
    int now = 0;
    if (p.lds) {
        int n2 = 2;
        while (n2 < rows) n2 *= 2;
        const unsigned zero = (unsigned)(ceil_div(V, 4096) < 256 ? ceil_div(V, 4096) : 256);
        hipLaunchKernelGGL((embed_sort_lds_kernel<I>), dim3(1 + zero), dim3(1024), (size_t)n2 * 8, st, id, (int)rows, n2, V, pad, key[0], pos[0], last);
        TOK_TRY(hipGetLastError());
    } else {
        // The first scatter marks the tokens that occur; from then on 512 workgroups more per launch clear the others' rows
        // (32768 x 2048 bf16 over 64000 tokens).
        const int64_t launches = 2 * (p.passes - 1);
        for (int q = 0; q < p.passes; ++q) {
            const I *src = q == 0 ? id : nullptr;
            EmbFill f[2] = {{last, (uint16_t *)out, 0, 0, d * (int64_t)(sizeof(T) / 2), p.nblk}, {last, (uint16_t *)out, 0, 0, d * (int64_t)(sizeof(T) / 2), p.nblk}};
            for (int h = 0; h < 2 && q > 0; ++h) {
                f[h].v0 = V * (2 * (q - 1) + h) / launches;
                f[h].v1 = V * (2 * (q - 1) + h + 1) / launches;
            }
            const unsigned grid = p.nblk + (q > 0 ? 512 : 0);
            hipLaunchKernelGGL((embed_hist_kernel<I>), dim3(grid), dim3(256), 0, st, src, key[now], rows, p.per_block, V, pad, 8 * q, hist, q == 0 ? last : nullptr, f[0]);
            TOK_TRY(hipGetLastError());
            hipLaunchKernelGGL((embed_scatter_kernel<I>), dim3(grid), dim3(256), 0, st, src, key[now], q == 0 ? nullptr : pos[now], rows, p.per_block, V, pad, 8 * q,
                               hist, key[now ^ 1], pos[now ^ 1], q == 0 && p.passes > 1 ? last : nullptr, f[1]);
            TOK_TRY(hipGetLastError());
            now ^= 1;
        }
    }
    const int tpr = pow2_at_least(ceil_div(d, 8), 8, 64);
    const int64_t ntile = ceil_div(d, (int64_t)tpr * 8), units = p.nchunk * ntile;
    auto sum = tpr == 8 ? embed_sum_kernel<T, 8> : tpr == 16 ? embed_sum_kernel<T, 16> : tpr == 32 ? embed_sum_kernel<T, 32> : embed_sum_kernel<T, 64>;
    hipLaunchKernelGGL(sum, dim3((unsigned)ceil_div(units, 256 / tpr)), dim3(256), 0, st, key[now], pos[now], rows, g, gs, (uint32_t)V, (int)d, scale, p.chunk, (int)ntile,
                       (T *)out, last, part);
    TOK_TRY(hipGetLastError());
    const int64_t joins = p.nchunk * (int64_t)p.jtile;
    const int64_t clear = p.passes > 1 ? 0 : V < JOIN_CLEAR ? V : JOIN_CLEAR;
    const EmbFill f = {last, (uint16_t *)out, 0, V, d * (int64_t)(sizeof(T) / 2), (int)joins};
    hipLaunchKernelGGL((embed_join_kernel<T>), dim3((unsigned)(joins + clear)), dim3(512), 0, st, key[now], last, rows, (uint32_t)V, part, p.chunk, p.jtile, (int)d, scale,
                       (T *)out, f);
    TOK_TRY(hipGetLastError());
    return 0;
}
template <class I>
__global__ __launch_bounds__(256) void embed_zero_kernel(I *out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = 0;
}
}  // namespace

#define EMB_DISPATCH(FN, ...)                                                                                     \
    (dtype == DNAG_F32 ? (ids_bytes == 8 ? FN<float, int64_t>(__VA_ARGS__) : FN<float, int32_t>(__VA_ARGS__))      \
     : dtype == DNAG_BF16 ? (ids_bytes == 8 ? FN<tbf16, int64_t>(__VA_ARGS__) : FN<tbf16, int32_t>(__VA_ARGS__))   \
                          : (ids_bytes == 8 ? FN<tf16, int64_t>(__VA_ARGS__) : FN<tf16, int32_t>(__VA_ARGS__)))

extern "C" int dnag_embed_forward(const void *ids, int ids_bytes, int64_t rows, const void *weight, int64_t weight_stride, int64_t num_tokens,
                                  int64_t dim, int dtype, float scale, void *out, void *stream) {
    if (int rc = check_embed(rows, num_tokens, dim, weight_stride, dtype, ids_bytes)) return rc;
    if (rows == 0) return 0;
    if (!ids || !weight || !out) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    return EMB_DISPATCH(forward_t, ids, rows, weight, weight_stride, num_tokens, dim, scale, out, (hipStream_t)stream);
}

extern "C" size_t dnag_embed_grad_workspace_bytes(int64_t rows, int64_t num_tokens, int64_t dim) {
    if (rows < 0 || rows > 0x7fffffffll || num_tokens < 1 || num_tokens > 0x7ffffffell || dim < 1 || dim > (1 << 20)) return 0;
    return grad_plan(rows, num_tokens, dim).bytes;
}

extern "C" int dnag_embed_grad(const void *ids, int ids_bytes, int64_t rows, const void *grad, int64_t grad_stride, int64_t num_tokens, int64_t dim,
                               int dtype, float scale, int64_t padding_idx, void *out, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_embed(rows, num_tokens, dim, grad_stride, dtype, ids_bytes)) return rc;
    if (!out || (rows > 0 && (!ids || !grad))) return dnag_fail(DNAG_E_ARG, "NULL pointer");
    hipStream_t st = (hipStream_t)stream;
    if (rows == 0) {                                   // no rows: a gradient of zeros
        const int64_t n = num_tokens * dim;
        const unsigned b = (unsigned)(ceil_div(n, 1024) < 4096 ? ceil_div(n, 1024) : 4096);
        if (dtype == DNAG_F32) hipLaunchKernelGGL((embed_zero_kernel<uint32_t>), dim3(b), dim3(256), 0, st, (uint32_t *)out, n);
        else hipLaunchKernelGGL((embed_zero_kernel<uint16_t>), dim3(b), dim3(256), 0, st, (uint16_t *)out, n);
        TOK_TRY(hipGetLastError());
        return 0;
    }
    const GradPlan p = grad_plan(rows, num_tokens, dim);
    // before anything is launched; the join's grid has the most lanes: 512 for 256 columns of a chunk, the sum's one for eight
    if (!p.few) if (int rc = grid_fits(p.nchunk * (int64_t)p.jtile + JOIN_CLEAR, 512)) return rc;
    if (workspace_bytes < p.bytes || (p.bytes && !workspace)) return dnag_fail(DNAG_E_WORKSPACE, "workspace has %zu bytes, %zu are needed", workspace_bytes, p.bytes);
    return EMB_DISPATCH(grad_t, p, ids, rows, grad, grad_stride, num_tokens, dim, scale, padding_idx, out, (char *)workspace, st);
}
