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

#include <type_traits>

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
// 127 2^(k-5): one more where the mantissa is above 0x7e0000.  From 2^-126 on, and up to 2^121, so that 127 2^e is finite (multiples
// beyond 127 are cut there: by less than a step).
__device__ __forceinline__ unsigned scale_byte(unsigned amax) { return (unsigned)min(max((int)((amax + 0x1ffffu) >> 23) - 6, 1), 248); }

__device__ __forceinline__ int quantise(float v, unsigned byte)
{
    if (!(fabsf(v) < INFINITY)) return -128;
    const float inverse = __uint_as_float((254u - byte) << 23);      // 2^-e: the exponent 127 - e
    return max(min(__float2int_rn(v * inverse), 127), -127);
}

// The kernels here move bytes.  A thread has 16 bytes of the tensor at a time, and loads several of them before it uses the first.
//
// Rows are cut into pieces of equal size (groups of 32 steps, or 16 bytes); those of all rows are counted through, and a CTA has kBlock of them, so that
// a piece's row is the CTA's first one or one of the next: found with 32-bit numbers.
struct Pieces {
    int64_t rows, T, G;
    int64_t each, all;           // pieces of a row, of all rows
    // 2^64 / each and 2^32 / each, rounded up (0 for 1): the upper half of a product is an exact quotient for numbers below 2^64 / each, or below
    // 4096 (each < 1024).  A division of 64 bits is 100 instructions, half of what 16 bytes take otherwise.
    uint64_t magic_far;
    unsigned magic;
};

template <int kBlock>
struct Place {
    static_assert(kBlock <= 1024, "a CTA's pieces");
    int64_t first, row0;         // of the CTA: piece, row
    unsigned rest0, here;        // which piece of its row the first one is; pieces
    __device__ __forceinline__ Place(const Pieces &s)
    {
        first = (int64_t)blockIdx.x * kBlock;
        row0 = s.magic_far ? (int64_t)__umul64hi((uint64_t)first, s.magic_far) : first;
        rest0 = (unsigned)(first - row0 * s.each);
        here = (unsigned)min(s.all - first, (int64_t)kBlock);
    }
    // rows from the CTA's first one, and which piece of its row the CTA's local-th one is
    __device__ __forceinline__ void operator()(const Pieces &s, unsigned local, unsigned &down, unsigned &piece) const
    {
        const unsigned r = rest0 + local, each = (unsigned)s.each;
        if (each >= 1024) down = r >= each;
        else down = s.magic ? __umulhi(r, s.magic) : r;
        piece = r - down * each;
    }
};

// 16 bytes a thread: kLanes of them have a group.  L: steps of a load, 16 bytes of them where rows' steps lie on 16 bytes; rows of other lengths are
// loaded in as large pieces as divide them (a line's other pieces are in L1 by then: one by one 48 us, 64 x 2312 x 301; with a
// lane for each step of a group it was 142).
template <typename E> constexpr int kCompressUnroll = sizeof(E) == 4 ? 4 : 2;
template <typename E> constexpr int kCompressBlock = 256 / (32 * (int)sizeof(E) / 16) * kCompressUnroll<E>;

template <int BYTES> struct Load;
template <> struct Load<16> { using type = uint4; };
template <> struct Load<8> { using type = uint2; };
template <> struct Load<4> { using type = uint32_t; };
template <> struct Load<2> { using type = uint16_t; };

template <typename E, int L>
__global__ void __launch_bounds__(256, 6)
compress_kernel(int8_t *q, uint8_t *scale, const E *x, const Pieces s)
{
    constexpr int W = 16 / (int)sizeof(E), kLanes = 32 / W, kUnroll = kCompressUnroll<E>;
    using Part = typename Load<L * (int)sizeof(E)>::type;
    const Place<kCompressBlock<E>> place(s);
    const unsigned t = (threadIdx.x % kLanes) * W, T = (unsigned)s.T, pad = (unsigned)(s.G * kGroup - s.T), lane0 = threadIdx.x / kLanes;
    const E *const x0 = x + (place.row0 * s.T + place.rest0 * (int64_t)kGroup);        // (of the CTA's first group)
    int8_t *const q0 = q + place.first * kGroup;
    uint8_t *const scale0 = scale + place.row0;
    unsigned down[kUnroll], group[kUnroll];
    float v[kUnroll][W];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned local = u * (256 / kLanes) + lane0;
        place(s, local, down[u], group[u]);
        const E *p = x0 + (int)(local * kGroup + t - down[u] * pad);
        const unsigned at = group[u] * kGroup + t;
        const unsigned end = local < place.here ? T : 0;
        Part raw[W / L];
#pragma unroll
        for (int j = 0; j < W / L; ++j) {
            raw[j] = Part();
            if (at + j * L < end) raw[j] = __ldg(reinterpret_cast<const Part *>(p) + j);
        }
        const E *e = reinterpret_cast<const E *>(raw);
#pragma unroll
        for (int j = 0; j < W; ++j) v[u][j] = as_float<E>(e[j]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned local = u * (256 / kLanes) + lane0;
        float largest = 0.0f;        // of magnitudes, some sign, NaN if one is
#pragma unroll
        for (int j = 0; j < W; ++j) asm("max.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(largest) : "f"(v[u][j]));
        unsigned top = __float_as_uint(largest) & 0x7fffffffu;
#pragma unroll
        for (int d = kLanes / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(~0u, top, d));
        unsigned byte, out[W / 4];
        if (!__any_sync(~0u, top >= 0x7e800000u)) {
            // whole multiples by adding 1.5 2^23, in whose last byte they are then: rounded to nearest, ties to even
            byte = (unsigned)max((int)((top + 0x1ffffu) >> 23) - 6, 1);
            const float inverse = __uint_as_float((254u - byte) << 23);
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                unsigned n[4];
#pragma unroll
                for (int l = 0; l < 4; ++l) n[l] = __float_as_uint(fmaf(v[u][j + l], inverse, 12582912.0f));
                out[j / 4] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
            }
        } else {
            // something large, or not finite
            top = 0;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const unsigned bits = __float_as_uint(v[u][j]) & 0x7fffffffu;
                top = max(top, bits < 0x7f800000u ? bits : 0u);
            }
#pragma unroll
            for (int d = kLanes / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(~0u, top, d));
            byte = scale_byte(top);
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                out[j / 4] = 0;
#pragma unroll
                for (int l = 0; l < 4; ++l) out[j / 4] |= (unsigned)(quantise(v[u][j + l], byte) & 0xff) << (8 * l);
            }
        }
        if (local < place.here) {
            unsigned *to = reinterpret_cast<unsigned *>(q0 + (local * kGroup + t));
            if (W == 4) to[0] = out[0];
            else *reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[W / 4 - 1]);
            if (t == 0) scale0[(int64_t)group[u] * s.rows + down[u]] = (uint8_t)byte;
        }
    }
}

// 16 bytes of a tensor that is read from 8 bits: W steps of a row from t on, some of them before its first or behind its last where rows do not lie
// on 16 bytes (not LINED).
template <int W>
struct Kept {
    static constexpr int kWords = W / 4 + 1;
    uint32_t word[kWords];
    unsigned byte, next;         // scales of the first step's group and of the one after it

    // q and scale of the CTA's first row; down: rows from there
    template <bool LINED>
    __device__ __forceinline__ void load(const uint32_t *q, const uint8_t *scale, const Pieces &s, unsigned down, int t)
    {
        const int words = (int)s.G * (kGroup / 4), at = t >> 2;
        const uint32_t *const p = q + down * (unsigned)words;
        if (LINED && W == 8) {
            const uint2 two = __ldg(reinterpret_cast<const uint2 *>(p + at));
            word[0] = two.x;
            word[1] = two.y;
        } else {
#pragma unroll
            for (int k = 0; k < (LINED ? W / 4 : kWords); ++k) word[k] = __ldg(p + (LINED ? at + k : min(max(at + k, 0), words - 1)));
        }
        const int group = (LINED ? t : max(t, 0)) >> 5;
        const uint8_t *const g = scale + ((int64_t)group * s.rows + down);
        byte = __ldg(g);
        if (!LINED) next = t > 0 && (t & 31) > 32 - W && group + 1 < (int)s.G ? __ldg(g + s.rows) : byte;
    }
    template <bool LINED>
    __device__ __forceinline__ void restore(float (&v)[W], int t) const
    {
        constexpr float kBias = 8388608.0f + 128.0f;
        const float s0 = __uint_as_float(byte << 23);
        uint32_t w[W / 4], none = 0;
#pragma unroll
        for (int k = 0; k < W / 4; ++k) {
            w[k] = (LINED ? word[k] : __funnelshift_r(word[k], word[k + 1], (t & 3) * 8)) ^ 0x80808080u;       // q + 128
            none |= (w[k] - 0x01010101u) & ~w[k];                                                             // a byte of 0: q is -128
        }
        if (!(none & 0x80808080u) && max(byte, LINED ? 0u : next) < 220u) {
            // 2^23 + q + 128 is the float that ends in that byte; times the scale, minus (2^23 + 128) times it: exact
            const float c0 = -kBias * s0;
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] = fmaf(__uint_as_float(__byte_perm(w[j / 4], 0x4b000000u, 0x7540 | (j % 4))), s0, c0);
            if (!LINED && next != byte) {
                const float s1 = __uint_as_float(next << 23), c1 = -kBias * s1;
#pragma unroll
                for (int j = 1; j < W; ++j)
                    if ((t & 31) + j >= 32) v[j] = fmaf(__uint_as_float(__byte_perm(w[j / 4], 0x4b000000u, 0x7540 | (j % 4))), s1, c1);
            }
        } else {
            // something that was not finite, or products that would not be
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int q = (int)((w[j / 4] >> (8 * (j % 4))) & 0xff) - 128;
                v[j] = q == -128 ? __uint_as_float(0x7fc00000u) : (float)q * __uint_as_float((LINED || (t & 31) + j < 32 ? byte : next) << 23);
            }
        }
    }
};

template <typename E, bool LINED>
__device__ __forceinline__ void store_steps(E *p, int t, int T, const float (&v)[16 / sizeof(E)])
{
    constexpr int W = 16 / (int)sizeof(E);
    if (LINED || (t >= 0 && t + W <= T)) {
        uint4 raw;
        E *e = reinterpret_cast<E *>(&raw);
#pragma unroll
        for (int j = 0; j < W; ++j) e[j] = as_type<E>(v[j]);
        *reinterpret_cast<uint4 *>(p) = raw;
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (t + j >= 0 && t + j < T) p[j] = as_type<E>(v[j]);
    }
}

// (64 x 2312 x 300 back in fours 34 us, in twos 39; surrogate gradients of 64 x 512 x 1450 in fours 84, in twos 73)
constexpr int kRestoreUnroll = 4, kGradUnroll = 2;

// the u-th 16 bytes of a thread: rows from the CTA's first one, and the step that they begin with
template <int W, bool LINED, int kBlock>
__device__ __forceinline__ bool read_place(const Pieces &s, const Place<kBlock> &place, int u, unsigned &down, int &t)
{
    const unsigned local = u * 256 + threadIdx.x;
    unsigned piece;
    place(s, local, down, piece);
    t = (int)piece * W - (LINED ? 0 : (int)((((unsigned)place.row0 + down) * (unsigned)s.T) & (W - 1)));
    return local < place.here && t < (int)s.T;
}

template <typename E, bool LINED>
__global__ void __launch_bounds__(256)
restore_kernel(E *out, const int8_t *q, const uint8_t *scale, const Pieces s)
{
    constexpr int W = 16 / (int)sizeof(E);
    const Place<256 * kRestoreUnroll> place(s);
    E *const out0 = out + place.row0 * s.T;
    const uint32_t *const q0 = reinterpret_cast<const uint32_t *>(q) + place.row0 * (s.G * (kGroup / 4));
    const uint8_t *const scale0 = scale + place.row0;
    unsigned down[kRestoreUnroll];
    int t[kRestoreUnroll];
    bool there[kRestoreUnroll];
    Kept<W> kept[kRestoreUnroll];
#pragma unroll
    for (int u = 0; u < kRestoreUnroll; ++u) {
        there[u] = read_place<W, LINED>(s, place, u, down[u], t[u]);
        if (there[u]) kept[u].template load<LINED>(q0, scale0, s, down[u], t[u]);
    }
#pragma unroll
    for (int u = 0; u < kRestoreUnroll; ++u)
        if (there[u]) {
            float v[W];
            kept[u].template restore<LINED>(v, t[u]);
            // A float16 above 65024 is kept as 64 * 2^10, half a step beyond the largest one, which it comes back as.  (2^9 and less: 65024 at most)
            if (std::is_same<E, __half>::value && max(kept[u].byte, LINED ? 0u : kept[u].next) >= 127 + 10) {
#pragma unroll
                for (int j = 0; j < W; ++j) v[j] = fabsf(v[j]) == 65536.0f ? copysignf(65504.0f, v[j]) : v[j];
            }
            store_steps<E, LINED>(out0 + ((int)(down[u] * (unsigned)s.T) + t[u]), t[u], (int)s.T, v);
        }
}

// The surrogate gradient (as spike_grad.cu has it) on a membrane potential in 8 bits: g c exp(-|u - theta| / tau), c = scale / tau, the exponential as
// 2^(-|u - theta| k) with k = log2(e) / tau in two floats, so that the product is rounded once, as a division would be.  Exponentials
// below 1.2e-38 are zero.
template <bool LINED>
__global__ void __launch_bounds__(256)
spike_grad_8_kernel(float *out, const float *g, const int8_t *q, const uint8_t *scale, const Pieces s, float theta, float k, float k_rest, float c)
{
    const Place<256 * kGradUnroll> place(s);
    const float *const g0 = g + place.row0 * s.T;
    float *const out0 = out + place.row0 * s.T;
    const uint32_t *const q0 = reinterpret_cast<const uint32_t *>(q) + place.row0 * (s.G * (kGroup / 4));
    const uint8_t *const scale0 = scale + place.row0;
    const int T = (int)s.T;
    int at[kGradUnroll], t[kGradUnroll];
    bool there[kGradUnroll];
    Kept<4> kept[kGradUnroll];
    float4 gv[kGradUnroll];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
        unsigned down;
        there[u] = read_place<4, LINED>(s, place, u, down, t[u]);
        at[u] = (int)(down * (unsigned)T) + t[u];
        if (!there[u]) continue;
        kept[u].template load<LINED>(q0, scale0, s, down, t[u]);
        const float *p = g0 + at[u];
        if (LINED || (t[u] >= 0 && t[u] + 4 <= T)) {
            gv[u] = *reinterpret_cast<const float4 *>(p);
        } else {
            gv[u].x = t[u] >= 0 ? p[0] : 0.0f;
            gv[u].y = t[u] + 1 >= 0 && t[u] + 1 < T ? p[1] : 0.0f;
            gv[u].z = t[u] + 2 >= 0 && t[u] + 2 < T ? p[2] : 0.0f;
            gv[u].w = t[u] + 3 < T ? p[3] : 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
        if (there[u]) {
            float v[4];
            const float up[4] = {gv[u].x, gv[u].y, gv[u].z, gv[u].w};
            kept[u].template restore<LINED>(v, t[u]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float d = fabsf(v[j] - theta);
                float e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-fmaf(d, k, d * k_rest)));
                v[j] = up[j] * (c * e);
            }
            store_steps<float, LINED>(out0 + at[u], t[u], T, v);
        }
}

// ------------------------------------------------------------------------------------------------ host side
static bool known(int dtype) { return dtype == SLAYER_B200_F32 || dtype == SLAYER_B200_BF16 || dtype == SLAYER_B200_F16; }
static bool off_element(const void *p, int dtype) { return ((uintptr_t)p & (dtype == SLAYER_B200_F32 ? 3 : 1)) != 0; }

static int check_rows(const char *op, int64_t rows, int64_t T)
{
    SB200_REQUIRE(rows >= 0 && T >= 0, "%s: negative size", op);
    // (pieces x pieces of a row below 2^64: Place)
    SB200_REQUIRE(rows <= (int64_t)1 << 37 && T <= (int64_t)1 << 29 && rows <= ((int64_t)1 << 37) / (ceil_div(T + 1, kGroup) * kGroup), "%s: too many steps", op);
    return SLAYER_B200_OK;
}

static Pieces pieces_of(int64_t rows, int64_t T, int64_t each)
{
    const uint64_t far = each == 1 ? 0 : ~(uint64_t)0 / (uint64_t)each + 1;
    return {rows, T, ceil_div(T, kGroup), each, rows * each, far, each == 1 || each >= 1024 ? 0u : (unsigned)((((uint64_t)1 << 32) + each - 1) / each)};
}

template <typename E, int L>
static void run_compress(int8_t *q, uint8_t *scale, const void *x, int64_t rows, int64_t T, cudaStream_t st)
{
    if constexpr (L > 1)
        if (T % L != 0 || ((uintptr_t)x & (L * sizeof(E) - 1)) != 0) return run_compress<E, L / 2>(q, scale, x, rows, T, st);
    const Pieces s = pieces_of(rows, T, ceil_div(T, kGroup));
    compress_kernel<E, L><<<(unsigned)ceil_div(s.all, kCompressBlock<E>), 256, 0, st>>>(q, scale, (const E *)x, s);
}

template <typename E>
static void run_restore(void *out, const int8_t *q, const uint8_t *scale, int64_t rows, int64_t T, cudaStream_t st)
{
    constexpr int W = 16 / (int)sizeof(E);
    const bool lined = T % W == 0;
    const Pieces s = pieces_of(rows, T, ceil_div(T + (lined ? 0 : W - 1), W));
    const unsigned blocks = (unsigned)ceil_div(s.all, 256 * kRestoreUnroll);
    if (lined) restore_kernel<E, true><<<blocks, 256, 0, st>>>((E *)out, q, scale, s);
    else restore_kernel<E, false><<<blocks, 256, 0, st>>>((E *)out, q, scale, s);
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
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == SLAYER_B200_F32) run_compress<float, 4>(q, scale, x, rows, T, st);
    else if (dtype == SLAYER_B200_BF16) run_compress<__nv_bfloat16, 8>(q, scale, x, rows, T, st);
    else run_compress<__half, 8>(q, scale, x, rows, T, st);
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
    SB200_REQUIRE(aligned16(out) && aligned16(q), "restore8: a pointer off its alignment");
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == SLAYER_B200_F32) run_restore<float>(out, q, scale, rows, T, st);
    else if (dtype == SLAYER_B200_BF16) run_restore<__nv_bfloat16>(out, q, scale, rows, T, st);
    else run_restore<__half>(out, q, scale, rows, T, st);
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
    SB200_REQUIRE(aligned16(out) && aligned16(g) && aligned16(q), "spike_grad8: a pointer off its alignment");
    const cudaStream_t st = (cudaStream_t)stream;
    const double exact = 1.4426950408889634 / (double)tau;
    const float k = (float)exact, k_rest = (float)(exact - (double)k);
    const bool lined = T % 4 == 0;
    const Pieces s = pieces_of(rows, T, ceil_div(T + (lined ? 0 : 3), 4));
    const unsigned blocks = (unsigned)ceil_div(s.all, 256 * kGradUnroll);
    if (lined) spike_grad_8_kernel<true><<<blocks, 256, 0, st>>>(out, g, q, scale_bytes, s, theta, k, k_rest, scale / tau);
    else spike_grad_8_kernel<false><<<blocks, 256, 0, st>>>(out, g, q, scale_bytes, s, theta, k, k_rest, scale / tau);
    return check_launch("spike_grad8 kernel launch");
}
