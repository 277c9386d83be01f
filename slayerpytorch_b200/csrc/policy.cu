// Losses of networks that answer with choices: rows of logits (spike counts, or a vocabulary's), one chosen entry each.
//
// With z = scale * x of a row, a the chosen entry and lp = z[a] - log sum_j exp(z[j]):
//   log-probability   lp, and d lp / d x[j] = scale * ((j == a) - p[j]),  p = softmax(z)
//   policy            per = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1),  r = exp(lp - old), d = ref - lp
//                     d per / d lp = -(r A where that is the smaller one) + kl (1 - exp(d))
//   preference        m_s = sum of a sequence's lp - ref_s,  h = beta (m_first - m_second),
//                     per pair (1 - e) log(1 + exp(-h)) + e log(1 + exp(h))
// What bounds the kernels is one read of the logits and one write of their gradient (HBM).  A row is read once from there: its running
// maximum and its sum of exponentials relative to that maximum are carried along (each thread's own, joined at the row's
// end), and the gradient is formed from a second read, out of the L2 cache, which holds the rows that are being worked on.  (Kept in shared
// memory instead, a row of 64 KB leaves room for three CTAs on an SM, not four: 4096 x 32768 bfloat16 115 us, read again 108.)
// A long row has a CTA of its own, a few of them on an SM: while one waits for its row's coefficient the others load.  Sums of
// exponentials are fp32 (each relative to the row's maximum, at most V terms of at most 1, added in a tree over the
// threads); what is said of one row - lp, the ratio, the loss - is computed in double, because a ratio that lies next to a
// border of the clip range decides whether the row has a gradient at all.  A double exponential takes as long as a quarter of a
// row's loads: the gradient waits for two of them, side by side in two lanes, and everything else that is said of
// a row comes in the launch that adds up the loss.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace sb200 {

enum RowMode { kLogProb, kPolicy, kGrad };

constexpr int kSums = 256;       // CTAs that add up a loss, at most

struct RowArgs {
    const void *logits;
    int64_t stride;               // elements between rows
    int64_t rows;
    int V;
    float scale, k;               // k = scale * log2(e)
    const int64_t *action;
    const uint8_t *mask;          // NULL: every row counts
    float *logp;                  // per row, may be NULL
    float2 *stats;                // per row: maximum of x, sum of exponentials
    // policy
    const float *old_lp, *ref_lp, *advantage;
    int64_t adv_len;              // rows per advantage
    double lo, hi, kl;            // clip range [lo, hi], weight of the KL term
    const int *counts;            // unmasked rows of each group of seq_len rows; NULL: share is the row's share
    int64_t seq_len;
    double share;                 // of a row; with counts: divided by the group's count
    double *gap;                  // kPolicy: (chosen - maximum) * scale, the part of lp that the sum does not give
    float *coef;                  // written by kPolicy; read by kGrad, where it may be NULL (1), one for each coef_len rows
    int64_t coef_len;
    const float *upstream;        // kGrad: one value, or one per row
    bool upstream_rows, only_if_not_one;
    void *grad;
    unsigned *arrived;            // kPolicy: set to zero for the sum that follows
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// 2^x to 2^-22 of itself, below 2^-126 zero: one instruction of the special function unit, where exp2f takes seven to
// keep results that are nothing beside a row's sum (what bounds a long row are instructions: 13 an entry with exp2f, 9 so)
__device__ __forceinline__ float two_to(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// sixteen bytes of a row
template <typename T>
struct Piece {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void open(float (&f)[N], uint4 v)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                f[i] = __uint_as_float(w[i]);
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                f[2 * i] = x.x;
                f[2 * i + 1] = x.y;
            }
        }
    }
    // of 16-bit entries: two of them, and the larger ones of two pairs
    static __device__ __forceinline__ void open2(float (&f)[2], uint32_t w)
    {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            f[0] = __uint_as_float(w << 16);
            f[1] = __uint_as_float(w & 0xffff0000u);
        } else {
            const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w));
            f[0] = x.x;
            f[1] = x.y;
        }
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
    {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 x = __hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
            return *reinterpret_cast<const uint32_t *>(&x);
        } else {
            const __half2 x = __hmax2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
            return *reinterpret_cast<const uint32_t *>(&x);
        }
    }
    static __device__ __forceinline__ uint4 close(const float (&f)[N])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(f[i]);
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&x);
            } else {
                const __half2 x = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&x);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// The exponentials of a part of a row with maximum m: 2^((x - base) k - c).  Near zero base is 0 and c = m k rounded: one multiply-add
// an entry.  That c is not m k exactly changes sums and the gradient's exponentials alike, and log_sum takes it out again.
// But the rounding of c grows with it (half a step is 2^-11 at 2^14 and 128 at 2^32, where 2^that is no float any more): where
// |m k| > 2^14, in rows that are filled with something or lie far from zero, base is m and c is 0, one instruction more an entry.
struct Frame {
    float base = 0.0f, c = 0.0f;
    __device__ __forceinline__ Frame(float m, float k)
    {
        c = __fmul_rn(m, k);
        if (!(fabsf(c) <= 16384.0f)) {
            base = m > -INFINITY ? m : 0.0f;           // (a part that holds only -inf has exponentials of 0, not of -inf + inf)
            c = 0.0f;
        }
    }
    __device__ __forceinline__ bool near() const { return base == 0.0f; }
    __device__ __forceinline__ float power(float x, float k) const { return two_to(fmaf(x - base, k, -c)); }
};

// Maximum and sum of exponentials of part of a row.
struct Soft {
    float m = -INFINITY, s = 0.0f;
    // the sum as one relative to n >= m, whose frame that of m becomes
    __device__ __forceinline__ void raise(float n, float k, Frame &f)
    {
        if (n == m) return;
        const Frame to(n, k);
        s *= m == -INFINITY ? 0.0f : two_to(fmaf(f.base - to.base, k, f.c - to.c));
        m = n;
        f = to;
    }
    __device__ __forceinline__ void raise(float n, float k)
    {
        Frame f(m, k);
        raise(n, k, f);
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N], float k)
    {
        float n = m;
#pragma unroll
        for (int i = 0; i < N; ++i) n = fmaxf(n, v[i]);
        raise(n, k);
        const Frame f(m, k);
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) t += f.power(v[i], k);
        s += t;
    }
    // a short row's elements, `step` apart; the frame of m is carried along (200000 x 500 float32 233 us; made anew an element 419)
    template <typename T>
    __device__ __forceinline__ void add_row(const T *x, int n, int step, float k, Frame &f)
    {
        for (int j = 0; j < n; j += step) {
            const float v = to_f(x[j]);
            raise(fmaxf(m, v), k, f);
            s += f.power(v, k);
        }
    }
    // pieces of a row: their maximum first, of 16-bit entries two at a time
    template <typename T, int NB>
    __device__ __forceinline__ void add(const uint4 (&v)[NB], float k)
    {
        using P = Piece<T>;
        float n = m;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int b = 0; b < NB; ++b) n = fmaxf(fmaxf(fmaxf(n, __uint_as_float(v[b].x)), fmaxf(__uint_as_float(v[b].y), __uint_as_float(v[b].z))), __uint_as_float(v[b].w));
        } else {
            uint32_t each[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) each[b] = P::larger(P::larger(v[b].x, v[b].y), P::larger(v[b].z, v[b].w));
            uint32_t top = each[0];
#pragma unroll
            for (int b = 1; b < NB; ++b) top = P::larger(top, each[b]);
            float both[2];
            P::open2(both, top);
            n = fmaxf(n, fmaxf(both[0], both[1]));
        }
        raise(n, k);
        const Frame f(m, k);
        float t[4] = {};
        if (f.near()) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float e[P::N];
                P::open(e, v[b]);
#pragma unroll
                for (int i = 0; i < P::N; ++i) t[i & 3] += two_to(fmaf(e[i], k, -f.c));
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float e[P::N];
                P::open(e, v[b]);
#pragma unroll
                for (int i = 0; i < P::N; ++i) t[0] += f.power(e[i], k);
            }
        }
        s += (t[0] + t[1]) + (t[2] + t[3]);
    }
    // all lanes of groups of G get the group's
    template <int G>
    __device__ __forceinline__ void meet(float k)
    {
        Frame f(m, k);
        meet<G>(k, f);
    }
    template <int G>
    __device__ __forceinline__ void meet(float k, Frame &f)
    {
        float n = m;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, o));
        raise(n, k, f);
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    // log of c's rounding: sum of exp((x - m) scale) = s exp(that)
    __device__ __forceinline__ static double rounding(float m, float k)
    {
        const Frame f(m, k);
        return f.near() && m > -INFINITY ? ((double)f.c - (double)m * (double)k) * 0.6931471805599453 : 0.0;
    }
    __device__ __forceinline__ static double log_sum(float m, float s, float k) { return log((double)s) + rounding(m, k); }
};

template <typename T>
__device__ __forceinline__ float chosen(const RowArgs &A, int64_t at, const T *x, int &a)
{
    a = at >= 0 && at < A.V ? (int)at : -1;
    return a < 0 ? NAN : to_f(x[a]);            // an action outside the row makes the row's results NaN
}

// A row's share of the loss
__device__ __forceinline__ double row_share(const RowArgs &A, int64_t row)
{
    if (!A.counts) return A.share;
    const int n = A.counts[(unsigned)row / (unsigned)A.seq_len];
    return A.share / (double)(n > 1 ? n : 1);
}

// The clipped term: its value at ratio r, and its derivative by lp
__device__ __forceinline__ double2 clipped(const RowArgs &A, double r, double gain)
{
    const double cut = (r < A.lo ? A.lo : r > A.hi ? A.hi : r) * gain, full = r * gain;
    return make_double2(-(full > cut ? cut : full), full > cut ? 0.0 : -full);
}

// What belongs to a row besides its logits: requested before they are read.
struct RowFacts {
    int a;                        // -1: outside the row
    float xa, old_lp, ref_lp, gain;
    double share;
};

template <RowMode MODE, typename T>
__device__ __forceinline__ RowFacts row_facts(const RowArgs &A, int64_t row, const T *x, int64_t action)
{
    RowFacts f = {};
    f.xa = chosen(A, action, x, f.a);
    if (MODE == kPolicy) {
        f.old_lp = A.old_lp[row];
        f.ref_lp = A.ref_lp ? A.ref_lp[row] : 0.0f;
        f.gain = A.advantage[(unsigned)row / (unsigned)A.adv_len];
        f.share = row_share(A, row);
    }
    return f;
}

// What one row comes to, from its maximum m and sum s.  Called by `lanes` together (lane: which of its row's); `write`: the first of
// these lanes stores the row's results.  Returns (c, c (1 / s)) to the first lane: the gradient is
// c * (j == a) - c (1 / s) * 2^((x[j] - base) k - c').
template <RowMode MODE>
__device__ __forceinline__ float2 row_result(const RowArgs &A, int64_t row, const RowFacts &f, float m, float s, int lane, unsigned lanes, bool write)
{
    float c = 0.0f;
    if constexpr (MODE == kGrad) {
        c = (A.coef ? A.coef[(unsigned)row / (unsigned)A.coef_len] : 1.0f) * (A.upstream_rows ? A.upstream[row] : A.upstream[0]) * A.scale;
    } else {
        const double gap = ((double)f.xa - (double)m) * (double)A.scale;
        write = write && lane == 0;
        if (write && A.stats) A.stats[row] = make_float2(m, s);
        if constexpr (MODE == kLogProb) {
            if (write) A.logp[row] = (float)(gap - Soft::log_sum(m, s, A.k));
        } else {
            // the first lane's is the ratio's exponential, the second's the KL term's
            const double e = exp(lane == 0 ? gap - (double)f.old_lp : (double)f.ref_lp - gap);
            const double off = Soft::rounding(m, A.k), sum = (double)s * (1.0 + off + 0.5 * off * off);      // |off| < 2^-11: exp(off) to 2e-11
            const double kl = A.ref_lp ? A.kl * (__shfl_down_sync(lanes, e, 1) * sum - 1.0) : 0.0;
            c = (float)(f.share * (clipped(A, e / sum, f.gain).y - kl));
            if (write) {
                A.gap[row] = gap;
                A.coef[row] = c;
            }
            c = c * 1.0f * A.scale;          // in the order of kGrad with an upstream of one: the same bits
        }
    }
    if (f.a < 0) c = NAN;
    return make_float2(c, c * (1.0f / s));
}

template <RowMode MODE>
__device__ __forceinline__ void masked_row(const RowArgs &A, int64_t row)
{
    if (MODE == kLogProb) A.logp[row] = 0.0f;
    if (MODE != kGrad && A.stats) A.stats[row] = make_float2(0.0f, 0.0f);
    if (MODE == kPolicy) A.coef[row] = 0.0f;
}

// ------------------------------------------------------------------------------------------- short rows
// G lanes per row
template <typename T, RowMode MODE, int G>
__global__ void __launch_bounds__(256) rows_short_kernel(RowArgs A)
{
    if (MODE == kGrad && A.only_if_not_one && A.upstream[0] == 1.0f) return;
    if (MODE == kPolicy && blockIdx.x == 0 && threadIdx.x == 0) *A.arrived = 0;
    const int lane = threadIdx.x % G;
    const int64_t step = (int64_t)gridDim.x * (256 / G);
    for (int64_t row0 = (int64_t)blockIdx.x * (256 / G); row0 < A.rows; row0 += step) {
        const int64_t row = row0 + threadIdx.x / G;
        const bool there = row < A.rows, live = there && !(A.mask && !A.mask[row]);
        const T *x = (const T *)A.logits + (live ? row : 0) * A.stride;
        T *g = A.grad && there ? (T *)A.grad + row * (int64_t)A.V : nullptr;
        RowFacts f = {};
        f.a = -1;
        if (live) f = row_facts<MODE>(A, row, x, A.action[row]);
        Soft soft;
        Frame frame(soft.m, A.k);
        if (MODE != kGrad) {
            if (live) soft.add_row(x + lane, A.V - lane, G, A.k, frame);
            __syncwarp();
            soft.meet<G>(A.k, frame);
        } else if (live) {
            const float2 st = A.stats[row];
            soft.m = st.x;
            soft.s = st.y;
            frame = Frame(st.x, A.k);
        }
        __syncwarp();
        float2 c = row_result<MODE>(A, live ? row : 0, f, soft.m, soft.s, lane, 0xffffffffu, live);
        if (!live && there && lane == 0) masked_row<MODE>(A, row);
        c.x = __shfl_sync(0xffffffffu, c.x, 0, G);
        c.y = __shfl_sync(0xffffffffu, c.y, 0, G);
        if (g)
            for (int j = lane; j < A.V; j += G)
                g[j] = from_f<T>(live ? fmaf(-c.y, frame.power(to_f(x[j]), A.k), j == f.a ? c.x : 0.0f) : 0.0f);
    }
}

// -------------------------------------------------------------------------------------------- long rows
// A CTA per row, or a cluster of them; each has its own stretch of the row, cut at 16-byte boundaries.
template <typename T, RowMode MODE>
__global__ void __launch_bounds__(512, 2) rows_long_kernel(RowArgs A)
{
    using P = Piece<T>;
    constexpr int N = P::N;
    __shared__ float2 part[16];          // the warps' maxima and sums
    __shared__ float2 whole;             // this CTA's (a cluster has one row)
    __shared__ float4 result;
    if (MODE == kGrad && A.only_if_not_one && A.upstream[0] == 1.0f) return;
    if (MODE == kPolicy && blockIdx.x == 0 && threadIdx.x == 0) *A.arrived = 0;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
    // a row each; or, where that costs less than more CTAs (launch_rows), several to a CTA alone
    for (int64_t row = blockIdx.x / C; row < A.rows; row += gridDim.x / C) {
        const T *x = (const T *)A.logits + row * A.stride;
        T *g = A.grad ? (T *)A.grad + row * (int64_t)A.V : nullptr;
        // the 16-byte pieces of the row, and the elements before and behind them
        const int head = min(A.V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
        const int pieces = (A.V - head) / N, per = (pieces + C - 1) / C;
        const int p0 = min(rank * per, pieces), p1 = min(p0 + per, pieces);
        const int tail0 = head + pieces * N;
        const uint4 *xp = (const uint4 *)(x + head);
        uint4 *gp = (uint4 *)(g + head);
        const bool wide = ((uintptr_t)gp & 15) == 0;
        const bool has_head = rank == 0 && tid < head, has_tail = rank == C - 1 && tail0 + tid < A.V;
        // a piece of the gradient: as one if it lies like the logits, else element by element
        const auto store = [&](int p, const float (&f)[N]) {
            if (wide) {
                __stcs(gp + p, P::close(f));
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) g[head + p * N + i] = from_f<T>(f[i]);
            }
        };
        const int64_t action = A.action[row];           // on its way while the mask is
        if (A.mask && !A.mask[row]) {
            if (rank == 0 && tid == 0) masked_row<MODE>(A, row);
            if (g) {
                const float zero[N] = {};
                for (int p = p0 + tid; p < p1; p += threads) store(p, zero);
                if (has_head) g[tid] = from_f<T>(0.0f);
                if (has_tail) g[tail0 + tid] = from_f<T>(0.0f);
            }
            continue;                        // the whole cluster
        }
        RowFacts f = {};
        if (warp == 0) f = row_facts<MODE>(A, row, x, action);
        Soft soft;
        if (MODE != kGrad) {
            int p = p0 + tid;
            for (; p + 7 * threads < p1; p += 8 * threads) {
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = xp[p + i * threads];
                soft.template add<T>(v, A.k);
            }
            for (; p + threads < p1; p += 2 * threads) {
                const uint4 v[2] = {xp[p], xp[p + threads]};
                soft.template add<T>(v, A.k);
            }
            if (p < p1) {
                const uint4 v[1] = {xp[p]};
                soft.template add<T>(v, A.k);
            }
            if (has_head) {
                const float v[1] = {to_f(x[tid])};
                soft.add(v, A.k);
            }
            if (has_tail) {
                const float v[1] = {to_f(x[tail0 + tid])};
                soft.add(v, A.k);
            }
            __syncwarp();
            soft.meet<32>(A.k);
            if (lane == 0) part[warp] = make_float2(soft.m, soft.s);
            __syncthreads();
            if (warp == 0) {
                soft = Soft();
                if (lane < threads / 32) {
                    soft.m = part[lane].x;
                    soft.s = part[lane].y;
                }
                soft.meet<16>(A.k);
            }
            if (C > 1) {
                if (tid == 0) whole = make_float2(soft.m, soft.s);
                cluster.sync();
                if (warp == 0) {
                    soft = Soft();
                    if (lane < C) {
                        const float2 o = *cluster.map_shared_rank(&whole, lane);
                        soft.m = o.x;
                        soft.s = o.y;
                    }
                    soft.meet<8>(A.k);
                }
            }
        } else if (warp == 0) {
            const float2 st = A.stats[row];
            soft.m = st.x;
            soft.s = st.y;
        }
        if (warp == 0 && lane < 2) {
            const float2 c = row_result<MODE>(A, row, f, soft.m, soft.s, lane, 3u, rank == 0);
            if (lane == 0) result = make_float4(c.x, c.y, soft.m, __int_as_float(f.a));
        }
        if (g) {
            __syncthreads();
            const float cx = result.x, cs = result.y;
            const Frame frame(result.z, A.k);
            const int a = __float_as_int(result.w);
            const auto value = [&](float v, float chosen) { return fmaf(-cs, frame.power(v, A.k), chosen); };
            const bool near = frame.near();
            const auto make = [&](int p, const uint4 &v) {
                float e[N];
                P::open(e, v);
                if (!near) {
#pragma unroll
                    for (int i = 0; i < N; ++i) e[i] = value(e[i], 0.0f);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) e[i] = -cs * two_to(fmaf(e[i], A.k, -frame.c));
                }
                store(p, e);
            };
            int p = p0 + tid;
            for (; p + 3 * threads < p1; p += 4 * threads) {
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = xp[p + i * threads];
#pragma unroll
                for (int i = 0; i < 4; ++i) make(p + i * threads, v[i]);
            }
            for (; p < p1; p += threads) make(p, xp[p]);
            // the chosen entry, behind its piece's own store
            const int pa = (a - head) / N;
            if (a >= head && pa >= p0 && pa < p1 && (pa - p0) % threads == tid) g[a] = from_f<T>(value(to_f(x[a]), cx));
            if (has_head) g[tid] = from_f<T>(value(to_f(x[tid]), tid == a ? cx : 0.0f));
            if (has_tail) g[tail0 + tid] = from_f<T>(value(to_f(x[tail0 + tid]), tail0 + tid == a ? cx : 0.0f));
        }
        if (gridDim.x < A.rows * C) __syncthreads();
    }
    if (C > 1) cluster.sync();           // no CTA leaves while another reads its sums
}

template <typename T, RowMode MODE>
int launch_rows(const RowArgs &A, cudaStream_t stream)
{
    const int64_t sms = sm_count();
    if (A.V <= 1024) {
        const bool eight = A.V <= 32;
        const int64_t blocks = ceil_div(A.rows, eight ? 32 : 8), cap = sms * 8;
        const unsigned grid = (unsigned)(blocks < cap ? blocks : cap);
        if (eight) rows_short_kernel<T, MODE, 8><<<grid, 256, 0, stream>>>(A);
        else rows_short_kernel<T, MODE, 32><<<grid, 256, 0, stream>>>(A);
        return check_launch("rows kernel launch");
    }
    const size_t bytes = (size_t)A.V * sizeof(T);
    // us with 128 / 256 / 512 threads (value and gradient): 20000 x 2048 bfloat16 107 / 164 / 298, 6000 x 8192 float32 87 / 97 / 144,
    // 3000 x 16384 float32 105 / 89, 4096 x 32768 bfloat16 144 / 122 / 144, 1505 x 50021 float32 191 / 167 / 146
    const int threads = bytes <= 32 * 1024 ? 128 : bytes <= 128 * 1024 ? 256 : 512;
    // CTAs per row: while there are SMs without one
    int C = 1;
    while (C < 8 && A.rows * C * 2 <= sms && (size_t)A.V / C > 8192) C *= 2;
    if (A.rows * C > 0x7fffffff) {
        set_error("%lld rows of %d entries", (long long)A.rows, A.V);
        return SLAYER_B200_EUNSUPPORTED;
    }
    auto kern = rows_long_kernel<T, MODE>;
    cudaLaunchConfig_t cfg = {};
    // a row each: with rows dealt out to resident CTAs, masked rows make some end early (4096 x 32768 bfloat16, a third of the rows
    // masked, 128 us, a row each 116 in the same build).  A gradient that may be there already should be told so to few CTAs.
    const int64_t cap = sms * 8 / C;
    cfg.gridDim = dim3((unsigned)((MODE == kGrad && A.only_if_not_one && A.rows > cap ? cap : A.rows) * C));
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, A);
    return check_launch("rows kernel launch");
}

template <RowMode MODE>
int launch_rows(int dtype, const RowArgs &A, cudaStream_t stream)
{
    switch (dtype) {
    case SLAYER_B200_F32: return launch_rows<float, MODE>(A, stream);
    case SLAYER_B200_BF16: return launch_rows<__nv_bfloat16, MODE>(A, stream);
    default: return launch_rows<__half, MODE>(A, stream);
    }
}

// ------------------------------------------------------------------------------------- sums and pairs
template <typename S>
__device__ __forceinline__ S block_sum(S v, S *part)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? part[lane] : S(0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// unmasked rows of each group of len rows
__global__ void __launch_bounds__(256) count_kernel(int *counts, const uint8_t *mask, int64_t len)
{
    __shared__ int part[32];
    const uint8_t *m = mask + blockIdx.x * len;
    int n = 0;
    for (int64_t i = threadIdx.x; i < len; i += blockDim.x) n += m[i] != 0;
    n = block_sum(n, part);
    if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// The loss, and the rows' log-probabilities: a thread has a row, the last CTA to come adds up the CTAs' sums in their order.
__global__ void __launch_bounds__(256) policy_sum_kernel(RowArgs A, float *loss, double *sums, unsigned *arrived)
{
    __shared__ double part[32];
    __shared__ bool last;
    double total = 0.0;
    for (int64_t row = blockIdx.x * 256ll + threadIdx.x; row < A.rows; row += gridDim.x * 256ll) {
        if (A.mask && !A.mask[row]) {
            if (A.logp) A.logp[row] = 0.0f;
            continue;
        }
        const float2 st = A.stats[row];
        const double lp = A.gap[row] - Soft::log_sum(st.x, st.y, A.k);
        if (A.logp) A.logp[row] = (float)lp;
        double per = clipped(A, exp(lp - (double)A.old_lp[row]), A.advantage[(unsigned)row / (unsigned)A.adv_len]).x;
        if (A.ref_lp) {
            const double d = (double)A.ref_lp[row] - lp;
            per += A.kl * (expm1(d) - d);
        }
        total += row_share(A, row) * per;
    }
    total = block_sum(total, part);
    if (threadIdx.x == 0) {
        sums[blockIdx.x] = total;
        __threadfence();
        last = atomicAdd(arrived, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    total = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) total += __ldcg(sums + i);
    total = block_sum(total, part);
    if (threadIdx.x == 0) *loss = (float)total;
}

// margin[s] = sum of a sequence's log-probabilities (masked ones are 0) - ref[s]
__global__ void __launch_bounds__(256) margin_kernel(double *margin, const float *logp, const float *ref, int64_t L)
{
    __shared__ double part[32];
    const float *lp = logp + blockIdx.x * L;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < L; i += blockDim.x) s += (double)lp[i];
    s = block_sum(s, part);
    if (threadIdx.x == 0) margin[blockIdx.x] = s - (double)ref[blockIdx.x];
}

// coef[s] = sum over the pairs that hold s of +- d loss / d h * beta, in the order of the pairs: a thread has a sequence, the
// CTA's threads work out 256 pairs at a time.  The first CTA adds up the loss.
__global__ void __launch_bounds__(256) pair_kernel(float *loss, float *coef, const double *margin, const int64_t *pairs,
                                                   int64_t S, int64_t P, double beta, double smoothing, double share)
{
    __shared__ double part[32];
    __shared__ int64_t first[256], second[256];
    __shared__ double slope[256];
    const int64_t me = blockIdx.x * 256ll + threadIdx.x;
    double mine = 0.0, total = 0.0;
    for (int64_t p0 = 0; p0 < P; p0 += 256) {
        const int64_t p = p0 + threadIdx.x;
        if (p < P) {
            const int64_t i = pairs[2 * p], j = pairs[2 * p + 1];
            const bool fine = i >= 0 && i < S && j >= 0 && j < S;    // another index makes the pair's loss and gradients NaN
            const double h = fine ? beta * (margin[i] - margin[j]) : (double)NAN;
            const double tail = log1p(exp(-fabs(h)));
            const double down = h < 0.0 ? -h : h > 0.0 ? 0.0 : h, up = h > 0.0 ? h : h < 0.0 ? 0.0 : h;    // max(-h, 0), max(h, 0)
            // (h has no bound where a choice is impossible: a term of weight 0 is 0 there too, and the slopes are the limits)
            total += share * ((smoothing < 1.0 ? (1.0 - smoothing) * (down + tail) : 0.0) + (smoothing > 0.0 ? smoothing * (up + tail) : 0.0));
            const double e = exp(-fabs(h)), sig = (h >= 0.0 ? 1.0 : e) / (1.0 + e);
            first[threadIdx.x] = i;
            second[threadIdx.x] = j;
            slope[threadIdx.x] = share * beta * (sig - (1.0 - smoothing));
        }
        __syncthreads();
        const int n = (int)(P - p0 < 256 ? P - p0 : 256);
        for (int i = 0; i < n; ++i) {
            if (first[i] == me) mine += slope[i];
            if (second[i] == me) mine -= slope[i];
        }
        __syncthreads();
    }
    if (me < S) coef[me] = (float)mine;
    if (blockIdx.x == 0) {
        total = block_sum(total, part);
        if (threadIdx.x == 0) *loss = (float)total;
    }
}

static int check_rows(const char *what, int dtype, int64_t rows, int64_t V, int64_t stride, double scale)
{
    SB200_REQUIRE(dtype == SLAYER_B200_F32 || dtype == SLAYER_B200_BF16 || dtype == SLAYER_B200_F16, "%s: unknown type %d", what, dtype);
    SB200_REQUIRE(rows >= 0 && V >= 1 && stride >= 0, "%s: bad size", what);
    SB200_REQUIRE(scale > 0.0 && scale < INFINITY, "%s: scale must be positive and finite", what);
    // scale log2(e), by which the exponents are multiplied, has to be an ordinary float32
    SB200_REQUIRE(scale >= 1.2e-38 && scale <= 2.3e38, "%s: scale must lie between 1.2e-38 and 2.3e38", what);
    if (V > (1 << 30) || rows > 0x7fffffff) {
        set_error("%s: %lld rows of %lld entries", what, (long long)rows, (long long)V);
        return SLAYER_B200_EUNSUPPORTED;
    }
    return SLAYER_B200_OK;
}

// logits and gradient at a multiple of their element, stats (read and written in pairs) at one of 8
static int check_places(const char *what, int dtype, const void *logits, const void *grad, const float *stats)
{
    const uintptr_t element = dtype == SLAYER_B200_F32 ? 3 : 1;
    SB200_REQUIRE((((uintptr_t)logits | (uintptr_t)grad) & element) == 0, "%s: logits and grad must be aligned to their elements", what);
    SB200_REQUIRE(((uintptr_t)stats & 7) == 0, "%s: stats must be aligned to 8 bytes", what);
    return SLAYER_B200_OK;
}

static RowArgs row_args(const void *logits, const int64_t *action, const uint8_t *mask, int64_t rows, int64_t V, int64_t stride, float scale)
{
    RowArgs A = {};
    A.logits = logits;
    A.stride = stride;
    A.rows = rows;
    A.V = (int)V;
    A.scale = scale;
    A.k = (float)((double)scale * 1.4426950408889634);
    A.action = action;
    A.mask = mask;
    return A;
}

}  // namespace sb200

using namespace sb200;

extern "C" int slayer_b200_log_prob(float *logp, float *stats, const void *logits, int dtype, const int64_t *action,
                                    const uint8_t *mask, int64_t rows, int64_t V, int64_t stride, float scale, void *stream)
{
    clear_error();
    int rc = check_rows("log_prob", dtype, rows, V, stride, scale);
    if (rc) return rc;
    if (rows == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(logp && logits && action, "log_prob: null pointer");
    rc = check_places("log_prob", dtype, logits, nullptr, stats);
    if (rc) return rc;
    RowArgs A = row_args(logits, action, mask, rows, V, stride, scale);
    A.logp = logp;
    A.stats = (float2 *)stats;
    return launch_rows<kLogProb>(dtype, A, (cudaStream_t)stream);
}

extern "C" int slayer_b200_logit_grad(void *grad, const void *logits, int dtype, const int64_t *action, const uint8_t *mask,
                                      const float *stats, const float *coef, int64_t coef_len, const float *upstream,
                                      int upstream_rows, int only_if_not_one, int64_t rows, int64_t V, int64_t stride, float scale,
                                      void *stream)
{
    clear_error();
    int rc = check_rows("logit_grad", dtype, rows, V, stride, scale);
    if (rc) return rc;
    if (rows == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(grad && logits && action && stats && upstream, "logit_grad: null pointer");
    SB200_REQUIRE(grad != logits, "logit_grad: grad must not alias logits");
    rc = check_places("logit_grad", dtype, logits, grad, stats);
    if (rc) return rc;
    SB200_REQUIRE(coef_len >= 1 && (!coef || rows % coef_len == 0), "logit_grad: rows must be whole groups of coef_len");
    RowArgs A = row_args(logits, action, mask, rows, V, stride, scale);
    A.stats = (float2 *)stats;
    A.coef = (float *)coef;
    A.coef_len = coef_len;
    A.upstream = upstream;
    A.upstream_rows = upstream_rows != 0;
    A.only_if_not_one = only_if_not_one && !upstream_rows;
    A.grad = grad;
    return launch_rows<kGrad>(dtype, A, (cudaStream_t)stream);
}

extern "C" int64_t slayer_b200_policy_loss_workspace(int64_t rows, int64_t seq_len)
{
    // what the sum does not give of each row, sums of the loss, a count, the sequences' counts
    return rows < 0 ? 0 : 8 * rows + 8 * kSums + 8 + 4 * (seq_len > 0 ? ceil_div(rows, seq_len) : 0);
}

extern "C" int slayer_b200_policy_loss(float *loss, void *grad, float *logp, float *stats, float *coef, void *workspace,
                                       const void *logits, int dtype, const int64_t *action, const float *old_logp, const float *advantage,
                                       int64_t adv_len, const float *ref_logp, const uint8_t *mask, int64_t rows, int64_t seq_len,
                                       int64_t V, int64_t stride, float scale, float clip_low, float clip_high, float kl, int reduction,
                                       void *stream)
{
    clear_error();
    int rc = check_rows("policy_loss", dtype, rows, V, stride, scale);
    if (rc) return rc;
    SB200_REQUIRE(loss, "policy_loss: null pointer");
    SB200_REQUIRE(clip_low >= 0.0f && clip_high >= 0.0f, "policy_loss: the clip range must not be negative");
    SB200_REQUIRE(reduction >= 0 && reduction <= 2, "policy_loss: unknown reduction %d", reduction);
    SB200_REQUIRE(adv_len >= 1 && rows % adv_len == 0, "policy_loss: rows must be whole groups of adv_len");
    SB200_REQUIRE(rows == 0 || (seq_len >= 1 && rows % seq_len == 0), "policy_loss: rows must be whole sequences");
    if (rows == 0) {
        if (cudaMemsetAsync(loss, 0, sizeof(float), (cudaStream_t)stream) != cudaSuccess) return check_launch("policy_loss");
        return SLAYER_B200_OK;
    }
    SB200_REQUIRE(coef && stats && workspace && logits && action && old_logp && advantage, "policy_loss: null pointer");
    SB200_REQUIRE(grad != logits, "policy_loss: grad must not alias logits");
    rc = check_places("policy_loss", dtype, logits, grad, stats);
    if (rc) return rc;
    SB200_REQUIRE(((uintptr_t)workspace & 7) == 0, "policy_loss: the workspace must be aligned to 8 bytes");
    const cudaStream_t st = (cudaStream_t)stream;
    RowArgs A = row_args(logits, action, mask, rows, V, stride, scale);
    A.logp = logp;
    A.stats = (float2 *)stats;
    A.old_lp = old_logp;
    A.ref_lp = ref_logp;
    A.advantage = advantage;
    A.adv_len = adv_len;
    A.lo = 1.0 - (double)clip_low;
    A.hi = 1.0 + (double)clip_high;
    A.kl = kl;
    A.coef = coef;
    A.coef_len = 1;
    A.gap = (double *)workspace;
    double *sums = A.gap + rows;
    unsigned *arrived = (unsigned *)(sums + kSums);
    A.arrived = arrived;
    A.grad = grad;
    const int64_t len = reduction == SLAYER_B200_MEAN ? rows : seq_len;
    A.share = reduction == SLAYER_B200_SUM ? 1.0 : 1.0 / (double)rows;     // without a mask all sequences are equally long
    if (reduction != SLAYER_B200_SUM && mask) {
        int *counts = (int *)(arrived + 2);
        SB200_REQUIRE(rows / len <= 0x7fffffff, "policy_loss: too many sequences");
        count_kernel<<<(unsigned)(rows / len), 256, 0, st>>>(counts, mask, len);
        rc = check_launch("count kernel launch");
        if (rc) return rc;
        A.counts = counts;
        A.seq_len = len;
        A.share = (double)len / (double)rows;          // 1, or 1 / sequences
    }
    rc = launch_rows<kPolicy>(dtype, A, st);
    if (rc) return rc;
    const int64_t blocks = ceil_div(rows, 256);
    policy_sum_kernel<<<(unsigned)(blocks < kSums ? blocks : kSums), 256, 0, st>>>(A, loss, sums, arrived);
    return check_launch("policy sum kernel launch");
}

extern "C" int64_t slayer_b200_preference_loss_workspace(int64_t sequences) { return sequences < 0 ? 0 : 8 * sequences + 8; }

extern "C" int slayer_b200_preference_loss(float *loss, float *coef, void *workspace, const float *logp, const float *ref_logp,
                                           const int64_t *pairs, int64_t sequences, int64_t seq_len, int64_t n_pairs, float beta,
                                           float smoothing, int reduction, void *stream)
{
    clear_error();
    SB200_REQUIRE(sequences >= 0 && seq_len >= 0 && n_pairs >= 0, "preference_loss: negative size");
    SB200_REQUIRE(reduction == SLAYER_B200_SUM || reduction == SLAYER_B200_MEAN, "preference_loss: unknown reduction %d", reduction);
    SB200_REQUIRE(smoothing >= 0.0f && smoothing <= 1.0f, "preference_loss: the smoothing must lie between 0 and 1");
    SB200_REQUIRE(loss, "preference_loss: null pointer");
    SB200_REQUIRE(sequences == 0 || (coef && workspace && ref_logp && (logp || seq_len == 0)), "preference_loss: null pointer");
    SB200_REQUIRE(n_pairs == 0 || pairs, "preference_loss: null pointer");
    SB200_REQUIRE(sequences <= 0x7fffffff, "preference_loss: too many sequences");
    SB200_REQUIRE(((uintptr_t)workspace & 7) == 0, "preference_loss: the workspace must be aligned to 8 bytes");
    const cudaStream_t st = (cudaStream_t)stream;
    double *margin = (double *)workspace;
    if (sequences > 0) {
        margin_kernel<<<(unsigned)sequences, 256, 0, st>>>(margin, logp, ref_logp, seq_len);
        int rc = check_launch("margin kernel launch");
        if (rc) return rc;
    }
    const double share = reduction == SLAYER_B200_MEAN && n_pairs ? 1.0 / (double)n_pairs : 1.0;
    pair_kernel<<<(unsigned)(sequences ? ceil_div(sequences, 256) : 1), 256, 0, st>>>(loss, coef, margin, pairs, sequences, n_pairs,
                                                                                     beta, smoothing, share);
    return check_launch("pair kernel launch");
}
