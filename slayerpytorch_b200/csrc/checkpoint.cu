// Tensors of a layer kept in 8 bits for its backward pass, and what that pass does with them.
//
// Each 32 consecutive steps of a row are whole multiples q, |q| <= 127, of a power of two: the smallest 2^e with max |x| <= 127 2^e.  So
// a value is off by at most 2^(e-1), 1/254 to 1/127 of the group's largest, and x 2^-e, its rounding and q 2^e are exact: the same
// input gives the same bits everywhere.  A power of two, because q 2^e is then a bfloat16 as it stands, which the weight gradient's
// matrix products take.  What is not finite is kept as -128 and comes back as NaN; it has no part in the scale.
//
// Layout: q [rows, 32 G] int8 with G = ceil(T / 32), zeros behind the last step; exponents [rows, G] as bytes e + 127.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace sb200 {

constexpr int kGroup = 32;

template <typename E> __device__ __forceinline__ float as_float(E v);
template <> __device__ __forceinline__ float as_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <typename E> __device__ __forceinline__ E as_type(float v);
template <> __device__ __forceinline__ float as_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half as_type<__half>(float v) { return __float2half_rn(v); }

// Byte of the scale for a largest magnitude given by its bits.  With amax = m 2^k, 1 <= m < 2: amax <= 127 2^(k-6) where m <= 127/64, else
// 127 2^(k-5).  From 2^-126 on, and up to 2^121, so that 127 2^e is finite (multiples beyond 127 are cut there: by less than a step).
__device__ __forceinline__ unsigned scale_byte(unsigned amax)
{
    const int e = (int)(amax >> 23) - 6 + ((amax & 0x7fffff) > 0x7e0000);
    return (unsigned)min(max(e, 1), 248);
}

__device__ __forceinline__ int quantise(float v, unsigned byte)
{
    if (!(fabsf(v) < INFINITY)) return -128;
    const float inverse = __uint_as_float((254u - byte) << 23);      // 2^-e: the exponent 127 - e
    return max(min(__float2int_rn(v * inverse), 127), -127);
}

__device__ __forceinline__ float restored(int q, unsigned byte)
{
    return q == -128 ? __uint_as_float(0x7fc00000u) : (float)q * __uint_as_float(byte << 23);
}

// a warp per group, a lane per step
template <typename E>
__global__ void __launch_bounds__(256)
compress_kernel(int8_t *q, uint8_t *scale, const E *x, int64_t groups_all, int64_t T, int64_t G)
{
    const int lane = threadIdx.x & 31;
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    if (group >= groups_all) return;
    const int64_t row = group / G, t = (group - row * G) * kGroup + lane;
    const float v = t < T ? as_float<E>(x[row * T + t]) : 0.0f;
    const unsigned bits = __float_as_uint(v) & 0x7fffffffu;
    const unsigned byte = scale_byte(__reduce_max_sync(~0u, bits < 0x7f800000u ? bits : 0u));
    q[group * kGroup + lane] = (int8_t)quantise(v, byte);
    if (lane == 0) scale[group] = (uint8_t)byte;
}

template <typename E>
__global__ void __launch_bounds__(256)
restore_kernel(E *out, const int8_t *q, const uint8_t *scale, int64_t groups_all, int64_t T, int64_t G)
{
    const int lane = threadIdx.x & 31;
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    if (group >= groups_all) return;
    const int64_t row = group / G, t = (group - row * G) * kGroup + lane;
    if (t < T) out[row * T + t] = as_type<E>(restored(q[group * kGroup + lane], scale[group]));
}

// the surrogate gradient (as spike_grad.cu has it) on a membrane potential in 8 bits
__global__ void __launch_bounds__(256)
spike_grad_8_kernel(float *out, const float *g, const int8_t *q, const uint8_t *scale, int64_t groups_all, int64_t T, int64_t G, float theta, float tau,
                    float c)
{
    const int lane = threadIdx.x & 31;
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    if (group >= groups_all) return;
    const int64_t row = group / G, t = (group - row * G) * kGroup + lane;
    if (t < T) out[row * T + t] = rho_times(g[row * T + t], restored(q[group * kGroup + lane], scale[group]), theta, tau, c);
}

// dW[o, i] = sum over samples n and steps t of g[n, o, t] x[n, i, t]: tiles of 64 x 64 outputs, 4 x 4 a thread; blockIdx.z takes every
// gridDim.z-th block of 32 steps, and the parts are added up in order behind it.
__global__ void __launch_bounds__(256)
weight_grad_kernel(float *part, const float *g, const int8_t *q, const uint8_t *scale, int64_t N, int64_t O, int64_t I, int64_t T, int64_t G)
{
    __shared__ float a[32][68], b[32][68];
    const int64_t o0 = (int64_t)blockIdx.y * 64, i0 = (int64_t)blockIdx.x * 64;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, step = threadIdx.x % 32;
    float acc[4][4] = {};
    for (int64_t k = blockIdx.z; k < N * G; k += gridDim.z) {
        const int64_t n = k / G, group = k - n * G, t = group * kGroup + step;
        for (int r = threadIdx.x / 32; r < 64; r += 8) {
            const int64_t o = o0 + r, i = i0 + r;
            a[step][r] = o < O && t < T ? g[(n * O + o) * T + t] : 0.0f;
            b[step][r] = i < I && t < T ? restored(q[((n * I + i) * G + group) * kGroup + step], scale[(n * I + i) * G + group]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 32; ++s) {
            float u[4], v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = a[s][ty * 4 + j], v[j] = b[s][tx * 4 + j];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int l = 0; l < 4; ++l) acc[j][l] = fmaf(u[j], v[l], acc[j][l]);
        }
        __syncthreads();
    }
    for (int j = 0; j < 4; ++j)
        for (int l = 0; l < 4; ++l) {
            const int64_t o = o0 + ty * 4 + j, i = i0 + tx * 4 + l;
            if (o < O && i < I) part[((int64_t)blockIdx.z * O + o) * I + i] = acc[j][l];
        }
}

__global__ void __launch_bounds__(256)
add_parts_kernel(float *out, const float *part, int64_t n, int parts)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    double sum = 0.0;
    for (int p = 0; p < parts; ++p) sum += (double)part[p * n + i];
    out[i] = (float)sum;
}

// ------------------------------------------------------------------------------------------------ host side
static bool known(int dtype) { return dtype == SLAYER_B200_F32 || dtype == SLAYER_B200_BF16 || dtype == SLAYER_B200_F16; }
static bool off_element(const void *p, int dtype) { return ((uintptr_t)p & (dtype == SLAYER_B200_F32 ? 3 : 1)) != 0; }

static int check_rows(const char *op, int64_t rows, int64_t T)
{
    SB200_REQUIRE(rows >= 0 && T >= 0, "%s: negative size", op);
    SB200_REQUIRE(rows <= (int64_t)1 << 40 && T <= (int64_t)1 << 40 && ceil_div(rows * ceil_div(T, kGroup), 8) <= 0x7fffffff, "%s: too many steps", op);
    return SLAYER_B200_OK;
}

static int64_t weight_parts(int64_t N, int64_t O, int64_t I, int64_t T)
{
    const int64_t tiles = ceil_div(O, 64) * ceil_div(I, 64), k = N * ceil_div(T, kGroup);
    int64_t parts = ceil_div((int64_t)sm_count() * 4, tiles);
    if (parts > k / 4) parts = k / 4;
    return parts < 1 ? 1 : (parts > 64 ? 64 : parts);
}

static int check_weight(const char *op, int64_t N, int64_t O, int64_t I, int64_t T)
{
    SB200_REQUIRE(N >= 0 && O >= 0 && I >= 0 && T >= 0, "%s: negative size", op);
    const int64_t most = (int64_t)1 << 31;
    SB200_REQUIRE(N < most && O <= 65535 * 64 && I < most && T < most && O * I < (int64_t)1 << 38 && N * ceil_div(T, kGroup) < (int64_t)1 << 40,
                  "%s: sizes are too large", op);
    return SLAYER_B200_OK;
}

}  // namespace sb200

extern "C" int slayer_b200_compress8(int8_t *q, uint8_t *scale, const void *x, int dtype, int64_t rows, int64_t T, void *stream)
{
    using namespace sb200;
    clear_error();
    SB200_REQUIRE(known(dtype), "compress8: unknown element type %d", dtype);
    const int rc = check_rows("compress8", rows, T);
    if (rc) return rc;
    if (rows == 0 || T == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(q && scale && x, "compress8: null pointer");
    SB200_REQUIRE(!off_element(x, dtype) && aligned16(q), "compress8: a pointer off its alignment");
    const int64_t G = ceil_div(T, kGroup), all = rows * G;
    const unsigned blocks = (unsigned)ceil_div(all, 8);
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == SLAYER_B200_F32) compress_kernel<float><<<blocks, 256, 0, st>>>(q, scale, (const float *)x, all, T, G);
    else if (dtype == SLAYER_B200_BF16) compress_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(q, scale, (const __nv_bfloat16 *)x, all, T, G);
    else compress_kernel<__half><<<blocks, 256, 0, st>>>(q, scale, (const __half *)x, all, T, G);
    return check_launch("compress8 kernel launch");
}

extern "C" int slayer_b200_restore8(void *out, const int8_t *q, const uint8_t *scale, int dtype, int64_t rows, int64_t T, void *stream)
{
    using namespace sb200;
    clear_error();
    SB200_REQUIRE(known(dtype), "restore8: unknown element type %d", dtype);
    const int rc = check_rows("restore8", rows, T);
    if (rc) return rc;
    if (rows == 0 || T == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(out && q && scale, "restore8: null pointer");
    SB200_REQUIRE(!off_element(out, dtype) && aligned16(q), "restore8: a pointer off its alignment");
    const int64_t G = ceil_div(T, kGroup), all = rows * G;
    const unsigned blocks = (unsigned)ceil_div(all, 8);
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == SLAYER_B200_F32) restore_kernel<float><<<blocks, 256, 0, st>>>((float *)out, q, scale, all, T, G);
    else if (dtype == SLAYER_B200_BF16) restore_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>((__nv_bfloat16 *)out, q, scale, all, T, G);
    else restore_kernel<__half><<<blocks, 256, 0, st>>>((__half *)out, q, scale, all, T, G);
    return check_launch("restore8 kernel launch");
}

extern "C" int slayer_b200_spike_grad8(float *out, const float *g, const int8_t *q, const uint8_t *scale_bytes, int64_t rows, int64_t T, float theta,
                                       float tau, float scale, void *stream)
{
    using namespace sb200;
    clear_error();
    const int rc = check_rows("spike_grad8", rows, T);
    if (rc) return rc;
    if (rows == 0 || T == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(out && g && q && scale_bytes, "spike_grad8: null pointer");
    SB200_REQUIRE(!off_element(out, SLAYER_B200_F32) && !off_element(g, SLAYER_B200_F32) && aligned16(q), "spike_grad8: a pointer off its alignment");
    const int64_t G = ceil_div(T, kGroup), all = rows * G;
    spike_grad_8_kernel<<<(unsigned)ceil_div(all, 8), 256, 0, (cudaStream_t)stream>>>(out, g, q, scale_bytes, all, T, G, theta, tau, scale / tau);
    return check_launch("spike_grad8 kernel launch");
}

extern "C" int64_t slayer_b200_weight_grad8_workspace(int64_t N, int64_t O, int64_t I, int64_t T)
{
    using namespace sb200;
    clear_error();
    const int rc = check_weight("weight_grad8_workspace", N, O, I, T);
    if (rc) return rc;
    if (N == 0 || O == 0 || I == 0 || T == 0) return 0;
    const int64_t parts = weight_parts(N, O, I, T);
    return parts > 1 ? parts * O * I * 4 : 0;
}

extern "C" int slayer_b200_weight_grad8(float *out, const float *g, const int8_t *q, const uint8_t *scale, int64_t N, int64_t O, int64_t I, int64_t T,
                                        void *workspace, void *stream)
{
    using namespace sb200;
    clear_error();
    const int rc = check_weight("weight_grad8", N, O, I, T);
    if (rc) return rc;
    if (O == 0 || I == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(out, "weight_grad8: null pointer");
    const cudaStream_t st = (cudaStream_t)stream;
    if (N == 0 || T == 0) {
        if (cudaMemsetAsync(out, 0, (size_t)(O * I) * 4, st) != cudaSuccess) return check_launch("weight_grad8 memset");
        return SLAYER_B200_OK;
    }
    SB200_REQUIRE(g && q && scale, "weight_grad8: null pointer");
    SB200_REQUIRE(!off_element(out, SLAYER_B200_F32) && !off_element(g, SLAYER_B200_F32) && aligned16(q), "weight_grad8: a pointer off its alignment");
    const int64_t parts = weight_parts(N, O, I, T);
    SB200_REQUIRE(parts == 1 || (workspace && aligned16(workspace)), "weight_grad8: the workspace must be aligned to 16 bytes");
    const dim3 grid((unsigned)ceil_div(I, 64), (unsigned)ceil_div(O, 64), (unsigned)parts);
    weight_grad_kernel<<<grid, 256, 0, st>>>(parts > 1 ? (float *)workspace : out, g, q, scale, N, O, I, T, ceil_div(T, kGroup));
    if (parts > 1) add_parts_kernel<<<(unsigned)ceil_div(O * I, 256), 256, 0, st>>>(out, (const float *)workspace, O * I, (int)parts);
    return check_launch("weight_grad8 kernel launch");
}
