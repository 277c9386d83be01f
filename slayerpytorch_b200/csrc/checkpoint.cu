// Tensors of a layer kept in 8 bits for its backward pass, and what that pass does with them.
//
// Each 32 consecutive steps of a row are whole multiples q, |q| <= 127, of a power of two: the smallest 2^e with max |x| <= 127 2^e.  So
// a value is off by at most 2^(e-1), 1/254 to 1/127 of the group's largest, and x 2^-e, its rounding and q 2^e are exact: the same
// input gives the same bits everywhere.  A power of two, because q 2^e is then a bfloat16 as it stands, which the weight gradient's
// matrix products take.  What is not finite is kept as -128 and comes back as NaN; it has no part in the scale.
//
// Layout: q [rows, 32 G] int8 with G = ceil(T / 32), zeros behind the last step; exponents [G, rows] as bytes e + 127 (the weight gradient's
// tiles take one group of steps of many rows).
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
    if (lane == 0) scale[(group - row * G) * (groups_all / G) + row] = (uint8_t)byte;
}

template <typename E>
__global__ void __launch_bounds__(256)
restore_kernel(E *out, const int8_t *q, const uint8_t *scale, int64_t groups_all, int64_t T, int64_t G)
{
    const int lane = threadIdx.x & 31;
    const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
    if (group >= groups_all) return;
    const int64_t row = group / G, t = (group - row * G) * kGroup + lane;
    if (t < T) out[row * T + t] = as_type<E>(restored(q[group * kGroup + lane], scale[(group - row * G) * (groups_all / G) + row]));
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
    if (t < T) out[row * T + t] = rho_times(g[row * T + t], restored(q[group * kGroup + lane], scale[(group - row * G) * (groups_all / G) + row]), theta, tau, c);
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
