// Orthogonalised updates: a matrix is brought near the orthogonal factor of its polar decomposition by Newton-Schulz products.
//
//   X0 = u / (|u|_F + eps),   X <- a X + (b A + c A A) X,  A = X X^T     (steps times; of a tall matrix, the transpose)
// Every step takes each singular value s to a s + b s^3 + c s^5, so they all end near one while the singular vectors stay.
// An optimiser step takes u from a gradient and its momentum and applies the result to the weight:
//   mom <- mu mom + g,   u = g + mu mom (or mom),   w <- w (1 - lr decay) - lr scale X
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <math.h>

#include "common.cuh"

namespace sb200 {

constexpr int kMaxJobs = 48;         // matrices per launch
constexpr int kNormParts = 64;       // partial sums of squares per matrix

struct NsJob {
    const void *src;                 // gradient, or the matrix itself
    float *mom;                      // NULL: the matrix itself is made orthogonal
    void *dst;                       // weight (updated), or the result
    int rows, cols, m, n;            // as stored; m <= n: as worked on
    float keep, step;                // w <- keep w - step X
    double *parts;
    float *x[2], *a, *b;
};

struct NsArgs {
    NsJob job[kMaxJobs];
    int jobs;
    float mu, ca, cb, cc, eps;
    bool nesterov;
};

template <typename T> __device__ __forceinline__ float ns_in(T v);
template <> __device__ __forceinline__ float ns_in(float v) { return v; }
template <> __device__ __forceinline__ float ns_in(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float ns_in(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T ns_out(float v);
template <> __device__ __forceinline__ float ns_out(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 ns_out(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half ns_out(float v) { return __float2half_rn(v); }

template <typename S>
__device__ __forceinline__ S ns_block_sum(S v, S *part)
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

// momentum, and the squares' partial sums (double: a sum over up to 2^31 squares, of values of any size)
template <typename T>
__global__ void __launch_bounds__(256) ns_momentum_kernel(const __grid_constant__ NsArgs A)
{
    __shared__ double part[32];
    const NsJob &J = A.job[blockIdx.y];
    const int64_t count = (int64_t)J.rows * J.cols;
    const T *g = (const T *)J.src;
    double sq = 0.0;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
        float u = ns_in(g[i]);
        if (J.mom) {
            const float m = fmaf(A.mu, J.mom[i], u);
            J.mom[i] = m;
            u = A.nesterov ? fmaf(A.mu, m, u) : m;
        }
        sq += (double)u * (double)u;
    }
    sq = ns_block_sum(sq, part);
    if (threadIdx.x == 0) J.parts[blockIdx.x] = sq;
}

template <typename T>
__global__ void __launch_bounds__(256) ns_normalise_kernel(const __grid_constant__ NsArgs A)
{
    const NsJob &J = A.job[blockIdx.y];
    double sq = 0.0;
    for (int i = 0; i < kNormParts; ++i) sq += J.parts[i];
    const float inv = (float)(1.0 / (sqrt(sq) + (double)A.eps));
    const int64_t count = (int64_t)J.rows * J.cols;
    const T *g = (const T *)J.src;
    const bool tall = J.rows > J.cols;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
        float u = ns_in(g[i]);
        if (J.mom) u = A.nesterov ? fmaf(A.mu, J.mom[i], u) : J.mom[i];
        const int64_t r = i / J.cols, c = i - r * J.cols;
        J.x[0][tall ? c * J.n + r : i] = u * inv;
    }
}

// PHASE 0: a = x x^T;  1: b = cb a + cc a a;  2: x' = ca x + b x.  One thread per element of a 16 x 16 tile.
template <int PHASE>
__global__ void __launch_bounds__(256) ns_product_kernel(const __grid_constant__ NsArgs A, int from)
{
    __shared__ float p[16][17], q[16][17];
    const NsJob &J = A.job[blockIdx.z];
    const int cols = PHASE == 2 ? J.n : J.m, K = PHASE == 0 ? J.n : J.m;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int i0 = blockIdx.y * 16, j0 = blockIdx.x * 16;
    if (i0 >= J.m || j0 >= cols) return;
    const float *x = J.x[from], *left = PHASE == 0 ? x : PHASE == 1 ? J.a : J.b;
    float s = 0.0f;
    for (int k0 = 0; k0 < K; k0 += 16) {
        p[ty][tx] = i0 + ty < J.m && k0 + tx < K ? left[(int64_t)(i0 + ty) * K + k0 + tx] : 0.0f;
        if (PHASE == 0) q[tx][ty] = j0 + ty < J.m && k0 + tx < K ? x[(int64_t)(j0 + ty) * K + k0 + tx] : 0.0f;
        else q[ty][tx] = k0 + ty < K && j0 + tx < cols ? (PHASE == 1 ? J.a : x)[(int64_t)(k0 + ty) * cols + j0 + tx] : 0.0f;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) s = fmaf(p[ty][k], q[k][tx], s);
        __syncthreads();
    }
    if (i0 + ty >= J.m || j0 + tx >= cols) return;
    const int64_t at = (int64_t)(i0 + ty) * cols + j0 + tx;
    if (PHASE == 0) J.a[at] = s;
    if (PHASE == 1) J.b[at] = A.cb * J.a[at] + A.cc * s;
    if (PHASE == 2) J.x[from ^ 1][at] = fmaf(A.ca, x[at], s);
}

template <typename T>
__global__ void __launch_bounds__(256) ns_apply_kernel(const __grid_constant__ NsArgs A, int from)
{
    const NsJob &J = A.job[blockIdx.y];
    const int64_t count = (int64_t)J.rows * J.cols;
    T *w = (T *)J.dst;
    const bool tall = J.rows > J.cols;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
        const int64_t r = i / J.cols, c = i - r * J.cols;
        const float o = J.x[from][tall ? c * J.n + r : i];
        w[i] = ns_out<T>(J.mom ? fmaf(J.keep, ns_in(w[i]), -J.step * o) : o);
    }
}

static size_t ns_job_bytes(int64_t m, int64_t n)
{
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    return up(kNormParts * 8) + 2 * up(4 * (size_t)(m * n)) + 2 * up(4 * (size_t)(m * m));
}

static int64_t ns_take(NsJob &J, unsigned char *at)
{
    unsigned char *const start = at;
    const auto take = [&](size_t bytes) { unsigned char *p = at; at += (bytes + 255) / 256 * 256; return p; };
    J.parts = (double *)take(kNormParts * 8);
    for (int i = 0; i < 2; ++i) J.x[i] = (float *)take(4 * (size_t)J.m * J.n);
    J.a = (float *)take(4 * (size_t)J.m * J.m);
    J.b = (float *)take(4 * (size_t)J.m * J.m);
    return at - start;
}

template <typename T>
static int ns_run(const NsArgs &A, int steps, cudaStream_t st)
{
    int m = 1, n = 1;
    for (int j = 0; j < A.jobs; ++j) {
        m = A.job[j].m > m ? A.job[j].m : m;
        n = A.job[j].n > n ? A.job[j].n : n;
    }
    const dim3 each(kNormParts, A.jobs);
    ns_momentum_kernel<T><<<each, 256, 0, st>>>(A);
    ns_normalise_kernel<T><<<each, 256, 0, st>>>(A);
    const unsigned mt = (m + 15) / 16, nt = (n + 15) / 16;
    int from = 0;
    for (int s = 0; s < steps; ++s, from ^= 1) {
        ns_product_kernel<0><<<dim3(mt, mt, A.jobs), 256, 0, st>>>(A, from);
        ns_product_kernel<1><<<dim3(mt, mt, A.jobs), 256, 0, st>>>(A, from);
        ns_product_kernel<2><<<dim3(nt, mt, A.jobs), 256, 0, st>>>(A, from);
    }
    ns_apply_kernel<T><<<each, 256, 0, st>>>(A, from);
    return check_launch("Newton-Schulz kernel launch");
}

// Whether the steps keep singular values from [0, 1] and the polynomial's factors in the range that the products can hold: the
// scaled 16-bit parts take values of x up to 8, of a and b up to 16.
static bool ns_bounded(int steps, double a, double b, double c)
{
    double top = 1.001;
    for (int s = 0; s < steps; ++s) {
        double next = 0.0;
        for (int i = 0; i <= 64; ++i) {
            const double v = top * i / 64, v2 = v * v, factor = b * v2 + c * v2 * v2;
            if (!(fabs(factor) < 14.0 && v2 < 14.0)) return false;
            const double p = fabs(v * (a + factor));
            if (!(p < 1e3)) return false;
            next = p > next ? p : next;
        }
        top = next * 1.01;
        if (!(top < 3.5)) return false;
    }
    return true;
}

static int ns_check(const char *what, int dtype, int steps, double a, double b, double c, double eps)
{
    SB200_REQUIRE(dtype == SLAYER_B200_F32 || dtype == SLAYER_B200_BF16 || dtype == SLAYER_B200_F16, "%s: unknown type %d", what, dtype);
    SB200_REQUIRE(steps >= 1 && steps <= 100, "%s: 1 to 100 steps", what);
    SB200_REQUIRE(eps >= 0.0 && eps < INFINITY, "%s: eps must not be negative", what);
    SB200_REQUIRE(ns_bounded(steps, a, b, c), "%s: with these coefficients singular values grow past 3.5", what);
    return SLAYER_B200_OK;
}

static int ns_shape(const char *what, int64_t rows, int64_t cols)
{
    SB200_REQUIRE(rows >= 0 && cols >= 0, "%s: negative size", what);
    if ((rows < cols ? rows : cols) > 32768 || (rows > cols ? rows : cols) > (1 << 22) || rows * cols > (1ll << 31)) {
        set_error("%s: a matrix of %lld x %lld", what, (long long)rows, (long long)cols);
        return SLAYER_B200_EUNSUPPORTED;
    }
    return SLAYER_B200_OK;
}

static int ns_dispatch(const NsArgs &A, int dtype, int steps, cudaStream_t st)
{
    switch (dtype) {
    case SLAYER_B200_F32: return ns_run<float>(A, steps, st);
    case SLAYER_B200_BF16: return ns_run<__nv_bfloat16>(A, steps, st);
    default: return ns_run<__half>(A, steps, st);
    }
}

}  // namespace sb200

using namespace sb200;

extern "C" int64_t slayer_b200_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, int dtype)
{
    (void)dtype;
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    return (int64_t)ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows) * (batch < kMaxJobs ? batch : kMaxJobs);
}

extern "C" int slayer_b200_orthogonalize(void *out, const void *in, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
                                         float a, float b, float c, float eps, void *workspace, void *stream)
{
    clear_error();
    int rc = ns_check("orthogonalize", dtype, steps, a, b, c, eps);
    if (rc) return rc;
    SB200_REQUIRE(batch >= 0, "orthogonalize: negative size");
    rc = ns_shape("orthogonalize", rows, cols);
    if (rc) return rc;
    if (batch == 0 || rows == 0 || cols == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(out && in && workspace, "orthogonalize: null pointer");
    SB200_REQUIRE(((uintptr_t)workspace & 255) == 0, "orthogonalize: the workspace must be aligned to 256 bytes");
    const size_t bytes = (size_t)rows * cols * (dtype == SLAYER_B200_F32 ? 4 : 2);
    for (int64_t first = 0; first < batch; first += kMaxJobs) {
        NsArgs A = {};
        A.jobs = (int)(batch - first < kMaxJobs ? batch - first : kMaxJobs);
        A.ca = a;
        A.cb = b;
        A.cc = c;
        A.eps = eps;
        unsigned char *at = (unsigned char *)workspace;
        for (int j = 0; j < A.jobs; ++j) {
            NsJob &J = A.job[j];
            J.src = (const unsigned char *)in + (first + j) * bytes;
            J.dst = (unsigned char *)out + (first + j) * bytes;
            J.rows = (int)rows;
            J.cols = (int)cols;
            J.m = (int)(rows < cols ? rows : cols);
            J.n = (int)(rows < cols ? cols : rows);
            at += ns_take(J, at);
        }
        rc = ns_dispatch(A, dtype, steps, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return SLAYER_B200_OK;
}

extern "C" int64_t slayer_b200_muon_step_workspace(const slayer_b200_muon_matrix *list, int64_t count, int dtype)
{
    (void)dtype;
    size_t most = 0, now = 0;
    int in = 0;
    for (int64_t i = 0; list && i < count; ++i) {
        const int64_t rows = list[i].rows, cols = list[i].cols;
        if (rows <= 0 || cols <= 0) continue;
        if (in++ == kMaxJobs) {
            in = 1;
            now = 0;
        }
        now += ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows);
        most = now > most ? now : most;
    }
    return (int64_t)most;
}

extern "C" int slayer_b200_muon_step(const slayer_b200_muon_matrix *list, int64_t count, int dtype, float lr, float momentum, int nesterov,
                                     float weight_decay, int adjust, int steps, float a, float b, float c, float eps, void *workspace,
                                     void *stream)
{
    clear_error();
    int rc = ns_check("muon_step", dtype, steps, a, b, c, eps);
    if (rc) return rc;
    SB200_REQUIRE(count >= 0, "muon_step: negative size");
    SB200_REQUIRE(count == 0 || list, "muon_step: null pointer");
    SB200_REQUIRE(adjust >= 0 && adjust <= 2, "muon_step: unknown adjustment %d", adjust);
    SB200_REQUIRE(((uintptr_t)workspace & 255) == 0, "muon_step: the workspace must be aligned to 256 bytes");
    for (int64_t i = 0; i < count; ++i) {
        const slayer_b200_muon_matrix &M = list[i];
        rc = ns_shape("muon_step", M.rows, M.cols);
        if (rc) return rc;
        SB200_REQUIRE(M.rows == 0 || M.cols == 0 || (M.weight && M.grad && M.momentum && workspace), "muon_step: null pointer");
    }
    int64_t i = 0;
    while (i < count) {
        NsArgs A = {};
        A.mu = momentum;
        A.nesterov = nesterov != 0;
        A.ca = a;
        A.cb = b;
        A.cc = c;
        A.eps = eps;
        unsigned char *at = (unsigned char *)workspace;
        for (; i < count && A.jobs < kMaxJobs; ++i) {
            const slayer_b200_muon_matrix &M = list[i];
            if (M.rows == 0 || M.cols == 0) continue;
            NsJob &J = A.job[A.jobs++];
            J.src = M.grad;
            J.mom = M.momentum;
            J.dst = M.weight;
            J.rows = (int)M.rows;
            J.cols = (int)M.cols;
            J.m = J.rows < J.cols ? J.rows : J.cols;
            J.n = J.rows < J.cols ? J.cols : J.rows;
            const double r = (double)J.rows / J.cols;
            const double factor = adjust == SLAYER_B200_MUON_SHAPE ? (r > 1.0 ? sqrt(r) : 1.0)
                                : adjust == SLAYER_B200_MUON_RMS   ? 0.2 * sqrt((double)J.n) : 1.0;
            J.keep = (float)(1.0 - (double)lr * (double)weight_decay);
            J.step = (float)((double)lr * factor);
            at += ns_take(J, at);
        }
        if (A.jobs == 0) break;
        rc = ns_dispatch(A, dtype, steps, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return SLAYER_B200_OK;
}
