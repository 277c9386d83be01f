// Losses of networks that answer with choices: rows of logits (spike counts, or a vocabulary's), one chosen entry each.
//
// With z = scale * x of a row, a the chosen entry and lp = z[a] - log sum_j exp(z[j]):
//   log-probability   lp, and d lp / d x[j] = scale * ((j == a) - p[j]),  p = softmax(z)
//   policy            per = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1),  r = exp(lp - old), d = ref - lp
//                     d per / d lp = -(r A where that is the smaller one) + kl (1 - exp(d))
//   preference        m_s = sum of a sequence's lp - ref_s,  h = beta (m_first - m_second),
//                     per pair (1 - e) log(1 + exp(-h)) + e log(1 + exp(h))
// What bounds the kernels is one read of the logits and one write of their gradient (HBM).  A row is read once: its running
// maximum and its sum of exponentials relative to that maximum are carried along (each thread's own, joined at the row's
// end), and the row itself waits in shared memory until its coefficient is known; the gradient is then formed from there.
// A thread keeps and takes back the 16-byte pieces that it loaded itself, so the copy needs no barrier.  Sums of
// exponentials are fp32 (each relative to the row's maximum, at most V terms of at most 1, added in a tree over the
// threads); what is said of one row - lp, the ratio, the loss - is computed in double, because a ratio that lies next to a
// border of the clip range decides whether the row has a gradient at all.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace sb200 {

enum RowMode { kLogProb, kPolicy, kGrad };

struct RowArgs {
    const void *logits;
    int64_t stride;               // elements between rows
    int64_t rows;
    int V;
    float scale, k;               // k = scale * log2(e)
    const int64_t *action;
    const uint8_t *mask;          // NULL: every row counts
    float *logp;                  // per row, may be NULL
    float2 *stats;                // per row: maximum of x, 1 / sum of exponentials
    // policy
    const float *old_lp, *ref_lp, *advantage;
    int64_t adv_len;              // rows per advantage
    double lo, hi, kl;            // clip range [lo, hi], weight of the KL term
    const int *counts;            // unmasked rows of each group of seq_len rows; NULL: share is the row's share
    int64_t seq_len;
    double share;                 // of a row; with counts: divided by the group's count
    double *row_loss;
    float *coef;                  // written by kPolicy; read by kGrad, where it may be NULL (1), one for each coef_len rows
    int64_t coef_len;
    const float *upstream;        // kGrad: one value, or one per row
    bool upstream_rows, only_if_not_one;
    void *grad;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

template <typename T>
struct alignas(16) Piece {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

// maximum and sum of exponentials of part of a row
struct Soft {
    float m = -INFINITY, s = 0.0f;
    // what the exponentials are taken relative to: of a part that holds only -inf, 0 (its exponentials are 0 then)
    __device__ __forceinline__ static float base(float m) { return m == -INFINITY ? 0.0f : m; }
    __device__ __forceinline__ void join(float om, float os, float k)
    {
        const float n = fmaxf(m, om), b = base(n);
        s = s * exp2f((m - b) * k) + os * exp2f((om - b) * k);
        m = n;
    }
    template <typename T, int N>
    __device__ __forceinline__ void add(const T (&v)[N], float k)
    {
        float n = m;
#pragma unroll
        for (int i = 0; i < N; ++i) n = fmaxf(n, to_f(v[i]));
        const float b = base(n);
        if (n != m) s *= exp2f((m - b) * k);
        m = n;
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) t += exp2f((to_f(v[i]) - b) * k);
        s += t;
    }
};

// What one row comes to: called by one thread with the row's maximum m and sum s.
// Returns (c, c (1 / s)): the gradient is c * (j == a) - c (1 / s) * exp2((x[j] - m) k).
// `write`: whether this thread is the one that stores the row's results.
template <RowMode MODE>
__device__ float2 row_result(const RowArgs &A, int64_t row, float m, float s, float xa, bool write)
{
    float c;
    if constexpr (MODE == kGrad) {
        c = (A.coef ? A.coef[row / A.coef_len] : 1.0f) * (A.upstream_rows ? A.upstream[row] : A.upstream[0]) * A.scale;
        return make_float2(c, c * s);          // s is 1 / sum here
    } else {
        const double lp = (double)(xa - m) * (double)A.scale - log((double)s);
        if (write) {
            if (A.logp) A.logp[row] = (float)lp;
            if (A.stats) A.stats[row] = make_float2(m, 1.0f / s);
        }
        if constexpr (MODE == kLogProb) return make_float2(0.0f, 0.0f);
        const double gain = A.advantage[row / A.adv_len];
        const double r = exp(lp - (double)A.old_lp[row]);
        const double cut = (r < A.lo ? A.lo : r > A.hi ? A.hi : r) * gain, full = r * gain;
        double per = -(full > cut ? cut : full), slope = full > cut ? 0.0 : -full;
        if (A.ref_lp) {
            const double d = (double)A.ref_lp[row] - lp, e = expm1(d);
            per += A.kl * (e - d);
            slope -= A.kl * e;
        }
        double share = A.share;
        if (A.counts) {
            const int n = A.counts[row / A.seq_len];
            share /= (double)(n > 1 ? n : 1);
        }
        c = (float)(share * slope);
        if (write) {
            A.row_loss[row] = share * per;
            A.coef[row] = c;
        }
        c = c * 1.0f * A.scale;          // in the order of kGrad with an upstream of one, and with its 1 / s: the same bits
        return make_float2(c, c * (1.0f / s));
    }
}

template <RowMode MODE>
__device__ void masked_row(const RowArgs &A, int64_t row)
{
    if (A.logp) A.logp[row] = 0.0f;
    if (MODE != kGrad && A.stats) A.stats[row] = make_float2(0.0f, 0.0f);
    if constexpr (MODE == kPolicy) {
        A.row_loss[row] = 0.0;
        A.coef[row] = 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ float chosen(const RowArgs &A, int64_t row, const T *x, int &a)
{
    const int64_t at = A.action[row];
    a = at >= 0 && at < A.V ? (int)at : -1;
    return a < 0 ? NAN : to_f(x[a]);            // an action outside the row makes the row's results NaN
}

// ------------------------------------------------------------------------------------------- short rows
// G lanes per row
template <typename T, RowMode MODE, int G>
__global__ void __launch_bounds__(256) rows_short_kernel(RowArgs A)
{
    if (MODE == kGrad && A.only_if_not_one && A.upstream[0] == 1.0f) return;
    const int lane = threadIdx.x % G;
    const int64_t step = (int64_t)gridDim.x * (256 / G);
    for (int64_t row0 = (int64_t)blockIdx.x * (256 / G); row0 < A.rows; row0 += step) {
        const int64_t row = row0 + threadIdx.x / G;
        const bool there = row < A.rows, live = there && !(A.mask && !A.mask[row]);
        const T *x = (const T *)A.logits + (live ? row : 0) * A.stride;
        T *g = A.grad && there ? (T *)A.grad + row * (int64_t)A.V : nullptr;
        Soft soft;
        if (MODE != kGrad) {
            if (live)
                for (int j = lane; j < A.V; j += G) {
                    const T v[1] = {x[j]};
                    soft.add(v, A.k);
                }
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) {
                const float om = __shfl_xor_sync(0xffffffffu, soft.m, o), os = __shfl_xor_sync(0xffffffffu, soft.s, o);
                soft.join(om, os, A.k);
            }
        } else if (live) {
            const float2 st = A.stats[row];
            soft.m = st.x;
            soft.s = st.y;
        }
        int a = -1;
        float2 c = make_float2(0.0f, 0.0f);
        if (live) {
            const float xa = chosen(A, row, x, a);
            if (lane == 0) {
                c = row_result<MODE>(A, row, soft.m, soft.s, xa, true);
                if (a < 0) c.x = c.y = NAN;
            }
        } else if (there && lane == 0) {
            masked_row<MODE>(A, row);
        }
        c.x = __shfl_sync(0xffffffffu, c.x, 0, G);
        c.y = __shfl_sync(0xffffffffu, c.y, 0, G);
        if (g)
            for (int j = lane; j < A.V; j += G)
                g[j] = from_f<T>(live ? (j == a ? c.x : 0.0f) - c.y * exp2f((to_f(x[j]) - soft.m) * A.k) : 0.0f);
    }
}

// -------------------------------------------------------------------------------------------- long rows
// A cluster of CTAs per row (often of one); each has its own stretch of the row, cut at 16-byte boundaries.
template <typename T, RowMode MODE, bool KEEP>
__global__ void __launch_bounds__(512) rows_long_kernel(RowArgs A)
{
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(16) unsigned char kept_bytes[];
    Piece<T> *kept = (Piece<T> *)kept_bytes;
    __shared__ float2 part[32];
    __shared__ float2 whole[2];          // this CTA's maximum and sum, by the row's parity
    __shared__ float4 result;
    if (MODE == kGrad && A.only_if_not_one && A.upstream[0] == 1.0f) return;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
    int parity = 0;
    for (int64_t row = blockIdx.x / C; row < A.rows; row += gridDim.x / C, parity ^= 1) {
        const T *x = (const T *)A.logits + row * A.stride;
        T *g = A.grad ? (T *)A.grad + row * (int64_t)A.V : nullptr;
        const bool live = !(A.mask && !A.mask[row]);
        // the 16-byte pieces of the row, and the elements before and behind them
        const int head = min(A.V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
        const int pieces = (A.V - head) / N, per = (pieces + C - 1) / C;
        const int p0 = min(rank * per, pieces), p1 = min(p0 + per, pieces);
        const int tail0 = head + pieces * N;
        const Piece<T> *xp = (const Piece<T> *)(x + head);
        if (!live) {
            if (rank == 0 && tid == 0) masked_row<MODE>(A, row);
            if (g) {
                if (rank == 0 && tid < head) g[tid] = from_f<T>(0.0f);
                if (rank == C - 1 && tail0 + tid < A.V) g[tail0 + tid] = from_f<T>(0.0f);
                const bool wide = ((uintptr_t)(g + head) & 15) == 0;
                Piece<T> zero;
#pragma unroll
                for (int i = 0; i < N; ++i) zero.v[i] = from_f<T>(0.0f);
                for (int p = p0 + tid; p < p1; p += threads) {
                    if (wide) ((Piece<T> *)(g + head))[p] = zero;
                    else
#pragma unroll
                        for (int i = 0; i < N; ++i) g[head + p * N + i] = zero.v[i];
                }
            }
            parity ^= 1;      // no exchange in this row
            continue;
        }
        Soft soft;
        if (MODE != kGrad) {
            int p = p0 + tid;
            for (; p + 3 * threads < p1; p += 4 * threads) {
                Piece<T> v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = xp[p + i * threads];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (KEEP) kept[p - p0 + i * threads] = v[i];
                    soft.add(v[i].v, A.k);
                }
            }
            for (; p < p1; p += threads) {
                const Piece<T> v = xp[p];
                if (KEEP) kept[p - p0] = v;
                soft.add(v.v, A.k);
            }
            if (rank == 0 && tid < head) {
                const T v[1] = {x[tid]};
                soft.add(v, A.k);
            }
            if (rank == C - 1 && tail0 + tid < A.V) {
                const T v[1] = {x[tail0 + tid]};
                soft.add(v, A.k);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float om = __shfl_xor_sync(0xffffffffu, soft.m, o), os = __shfl_xor_sync(0xffffffffu, soft.s, o);
                soft.join(om, os, A.k);
            }
            if (lane == 0) part[warp] = make_float2(soft.m, soft.s);
            __syncthreads();
            if (warp == 0) {
                soft = Soft();
                if (lane < threads / 32) {
                    soft.m = part[lane].x;
                    soft.s = part[lane].y;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const float om = __shfl_xor_sync(0xffffffffu, soft.m, o), os = __shfl_xor_sync(0xffffffffu, soft.s, o);
                    soft.join(om, os, A.k);
                }
                if (lane == 0) whole[parity] = make_float2(soft.m, soft.s);
            }
            if (C > 1) {
                cluster.sync();
                if (warp == 0) {
                    soft = Soft();
                    for (int r = 0; r < C; ++r) {
                        const float2 o = *cluster.map_shared_rank(&whole[parity], r);
                        soft.join(o.x, o.y, A.k);
                    }
                }
            }
        }
        if (tid == 0) {
            int a;
            const float xa = chosen(A, row, x, a);
            if (MODE == kGrad) {
                const float2 st = A.stats[row];
                soft.m = st.x;
                soft.s = st.y;
            }
            float2 c = make_float2(0.0f, 0.0f);
            if (rank == 0 || g) {
                c = row_result<MODE>(A, row, soft.m, soft.s, xa, rank == 0);    // the other CTAs need the coefficients too
                if (a < 0) c.x = c.y = NAN;
            }
            result = make_float4(c.x, c.y, soft.m, __int_as_float(a));
        }
        if (g) {
            __syncthreads();
            const float cx = result.x, cs = result.y, m = result.z;
            const int a = __float_as_int(result.w);
            auto value = [&](T v, int j) { return from_f<T>((j == a ? cx : 0.0f) - cs * exp2f((to_f(v) - m) * A.k)); };
            if (rank == 0 && tid < head) g[tid] = value(x[tid], tid);
            if (rank == C - 1 && tail0 + tid < A.V) g[tail0 + tid] = value(x[tail0 + tid], tail0 + tid);
            const bool wide = ((uintptr_t)(g + head) & 15) == 0;
            for (int p = p0 + tid; p < p1; p += threads) {
                const Piece<T> v = KEEP ? kept[p - p0] : xp[p];
                const int j = head + p * N;
                if (wide) {
                    Piece<T> o;
#pragma unroll
                    for (int i = 0; i < N; ++i) o.v[i] = value(v.v[i], j + i);
                    ((Piece<T> *)(g + head))[p] = o;
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) g[j + i] = value(v.v[i], j + i);
                }
            }
        }
        __syncthreads();                 // part, result
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
    const int threads = A.V <= 8192 ? 256 : 512;
    // CTAs per row: until the row's stretch fits the shared memory kept for it, and while there are SMs without one
    const size_t most = 100 * 1024;
    const size_t bytes = ((size_t)A.V * sizeof(T) + 15) / 16 * 16;
    int C = 1;
    while (C < 8 && (ceil_div(bytes, C) > (int64_t)most || (A.rows * C * 2 <= sms && (size_t)A.V / C > 8192))) C *= 2;
    const int64_t stretch = (ceil_div(bytes / 16, C) + 1) * 16;
    const bool keep = MODE == kPolicy && A.grad && stretch <= (int64_t)most;
    const size_t smem = keep ? (size_t)stretch : 0;
    auto kern = keep ? rows_long_kernel<T, MODE, MODE == kPolicy> : rows_long_kernel<T, MODE, false>;
    int rc = reserve_dynamic_smem((const void *)kern, smem);
    if (rc) return rc;
    const int64_t cap = sms * (threads == 256 ? 8 : 4) / C;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((A.rows < cap ? A.rows : cap) * C));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
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

__global__ void __launch_bounds__(1024) sum_kernel(float *out, const double *v, int64_t n)
{
    __shared__ double part[32];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += v[i];
    s = block_sum(s, part);
    if (threadIdx.x == 0) *out = (float)s;
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
            total += share * ((1.0 - smoothing) * (down + tail) + smoothing * (up + tail));
            const double e = exp(-fabs(h)), sig = (h >= 0.0 ? 1.0 : e) / (1.0 + e);
            first[threadIdx.x] = i;
            second[threadIdx.x] = j;
            slope[threadIdx.x] = share * beta * (sig - (1.0 - smoothing)) + 0.0 * h;
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
    if (V > (1 << 30)) {
        set_error("%s: rows of %lld entries", what, (long long)V);
        return SLAYER_B200_EUNSUPPORTED;
    }
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
    SB200_REQUIRE(coef_len >= 1, "logit_grad: coef_len must be at least 1");
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
    return rows < 0 ? 0 : 8 * rows + 4 * (seq_len > 0 ? ceil_div(rows, seq_len) : 0) + 16;
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
    SB200_REQUIRE(adv_len >= 1, "policy_loss: adv_len must be at least 1");
    SB200_REQUIRE(rows == 0 || (seq_len >= 1 && rows % seq_len == 0), "policy_loss: rows must be whole sequences");
    if (rows == 0) {
        if (cudaMemsetAsync(loss, 0, sizeof(float), (cudaStream_t)stream) != cudaSuccess) return check_launch("policy_loss");
        return SLAYER_B200_OK;
    }
    SB200_REQUIRE(coef && workspace && logits && action && old_logp && advantage, "policy_loss: null pointer");
    SB200_REQUIRE(grad != logits, "policy_loss: grad must not alias logits");
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
    A.row_loss = (double *)workspace;
    A.grad = grad;
    const int64_t len = reduction == SLAYER_B200_MEAN ? rows : seq_len;
    A.share = reduction == SLAYER_B200_SUM ? 1.0 : 1.0 / (double)rows;     // without a mask all sequences are equally long
    if (reduction != SLAYER_B200_SUM && mask) {
        int *counts = (int *)(A.row_loss + rows);
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
    sum_kernel<<<1, 1024, 0, st>>>(loss, A.row_loss, rows);
    return check_launch("sum kernel launch");
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
