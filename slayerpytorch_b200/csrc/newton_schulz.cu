// Orthogonalised updates: a matrix is brought near the orthogonal factor of its polar decomposition by Newton-Schulz products.
//
//   X0 = u / (|u|_F + eps),   X <- a X + (b A + c A A) X,  A = X X^T     (steps times; of a tall matrix, the transpose)
// Every step takes each singular value s to a s + b s^3 + c s^5, so they all end near one while the singular vectors stay.
// An optimiser step takes u from a gradient and its momentum and applies the result to the weight:
//   mom <- mu mom + g,   u = g + mu mom (or mom),   w <- w (1 - lr decay) - lr scale X
//
// The work is matrix products, m m n + m m m + 2 m m n multiply-adds a step for m <= n with the symmetric halves left out, so
// they run on the tensor cores, on 16-bit parts of the 32-bit values.  Everything has a known size - |X|_F <= 1 at the start, no
// singular value ever above 3.5 - so fp16 with a fixed power-of-two scale holds it, and holds 11 bits where bf16 holds 8.
//     v = hi + lo, two fp16 values, 22 bits and a sign;  v w ~ hi hi + hi lo + lo hi, the left out lo lo being 2^-24 of it.
// Three products instead of one, for bfloat16 matrices too: with hi alone, 11 bits, their results ended 1.2 to 2.2 times as far off as
// their own rounding to 8 bits (6 x 1023 x 2049 in 387 us instead of 715).
// Sums are fp32: those of 64 to 192 products in tensor memory, longer ones in registers (see NsTile::group).  Five steps end 0.2 to 0.7
// times as far off as with fp32 products; matrices that stay on the chip, whose fp32 sums are short, 0.6 to 1.9 times.
// Entries of X are held to 2^-37 at best (an fp16's smallest step over the scale): enough where the norm is not far below eps.
//
// X, A and B = b A + c A A live in the workspace as blocks of 128 x 64 elements, padded with zeros, each block laid out as the
// tensor core reads it from shared memory (tensor.cuh), hi before lo: every load is a contiguous copy of 8 to 32 KB, whatever
// the matrix's sizes, and one form of X serves both as rows (X X^T) and as columns (B X).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "tensor.cuh"

namespace sb200 {

constexpr int kMaxJobs = 48;         // matrices per launch,
constexpr int64_t kMostBytes = 4ll << 30;      // fewer where their workspace would pass this (one of 2300 x 2300 fills the SMs alone)
constexpr int kNormParts = 256;      // partial sums of squares per matrix
constexpr int kStatusNsTimeout = 0x5103;
constexpr int kWaitLimit = 1 << 22;
constexpr int kParts = 2;            // fp16 values that a value is kept as
constexpr int kBlock = 128 * 64 * 2; // bytes of a block
constexpr float kScaleX = 8192.0f, kScaleA = 4096.0f;      // of X; of A and B

struct NsJob {
    const void *src;                 // gradient, or the matrix itself
    float *mom;                      // NULL: the matrix itself is made orthogonal
    void *dst;                       // weight (updated), or the result
    int rows, cols, m, n;            // as stored; m <= n: as worked on
    float keep, step;                // w <- keep w - step X
    double *parts;
    int norm_parts;
    unsigned char *x[2], *a, *b;     // blocks: row blocks of 128, in each of them column blocks of 64
    int first[3];                    // this launch's first block of the passes over elements; first tile of the products (A, X)
};

struct NsArgs {
    NsJob job[kMaxJobs];
    int jobs;
    float mu, ca, cb, cc, eps;
    bool nesterov;
};

static __host__ __device__ __forceinline__ int ns_rb(int v) { return (v + 127) / 128; }            // row blocks
static __host__ __device__ __forceinline__ int ns_cb(int v) { return (v + 127) / 128 * 2; }        // column blocks

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

// the job that a block or tile belongs to: the last one that does not begin behind it
template <int WHICH>
__device__ __forceinline__ int ns_find(const NsArgs &A, int at)
{
    int j = 0;
    while (j + 1 < A.jobs && A.job[j + 1].first[WHICH] <= at) ++j;
    return j;
}

// What turns u into the scaled X0: one factor, or two where the norm is so small that its inverse is no float.
struct NsScale {
    float lift, inv;
    __device__ __forceinline__ NsScale(double squares, float eps)
    {
        const double norm = sqrt(squares) + (double)eps;
        lift = norm < 1e-25 ? 0x1p80f : 1.0f;
        inv = (float)((double)kScaleX / (norm * (double)lift));
    }
    __device__ __forceinline__ float operator()(float u) const { return u * lift * inv; }
};

__device__ __forceinline__ bool ns_wide(const void *p) { return ((uintptr_t)p & 15) == 0; }

// eight elements that follow one another, as 32-bit values
template <typename T>
__device__ __forceinline__ void ns_load8(float (&v)[8], const T *p)
{
    if constexpr (sizeof(T) == 4) {
        const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *(const uint4 *)p;
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t h = (uint16_t)(w[i >> 1] >> (i & 1) * 16);
            v[i] = ns_in(*reinterpret_cast<const T *>(&h));
        }
    }
}

// o, or keep w + o where a weight is updated, as 16 bytes
template <typename T>
__device__ __forceinline__ void ns_store16(T *at, const float (&o)[16 / sizeof(T)], const uint4 &w, float keep, bool update)
{
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    uint32_t out[4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __float_as_uint(update ? fmaf(keep, __uint_as_float(ws[i]), o[i]) : o[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint16_t h[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint16_t old = (uint16_t)(ws[i] >> 16 * e);
                const T x = ns_out<T>(update ? fmaf(keep, ns_in(*reinterpret_cast<const T *>(&old)), o[2 * i + e]) : o[2 * i + e]);
                h[e] = *reinterpret_cast<const uint16_t *>(&x);
            }
            out[i] = h[0] | (uint32_t)h[1] << 16;
        }
    }
    *(uint4 *)at = make_uint4(out[0], out[1], out[2], out[3]);
}

// momentum, and the squares' partial sums (double: a sum over up to 2^31 squares, of values of any size)
template <typename T>
__global__ void __launch_bounds__(256) ns_momentum_kernel(const __grid_constant__ NsArgs A, unsigned *arrived)
{
    if (blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;
    __shared__ double part[32];
    const NsJob &J = A.job[ns_find<0>(A, blockIdx.x)];
    const int me = blockIdx.x - J.first[0];
    const int64_t count = (int64_t)J.rows * J.cols, step = J.norm_parts * 256ll, start = me * 256ll + threadIdx.x;
    const T *g = (const T *)J.src;
    float *mom = J.mom;
    double sq = 0.0;
    int64_t done = 0;
    if (ns_wide(g) && ns_wide(mom)) {
        const int64_t eights = count / 8;
        done = eights * 8;
        constexpr int U = 2;                       // pieces requested before the first is used
        for (int64_t i0 = start; i0 < eights; i0 += U * step) {
            float u[U][8], m[U][8];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t i = i0 + k * step;
                if (i < eights) {
                    ns_load8(u[k], g + i * 8);
                    if (mom) ns_load8(m[k], mom + i * 8);
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t i = i0 + k * step;
                if (i < eights) {
                    if (mom) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            m[k][e] = fmaf(A.mu, m[k][e], u[k][e]);
                            u[k][e] = A.nesterov ? fmaf(A.mu, m[k][e], u[k][e]) : m[k][e];
                        }
                        *(float4 *)(mom + i * 8) = make_float4(m[k][0], m[k][1], m[k][2], m[k][3]);
                        *(float4 *)(mom + i * 8 + 4) = make_float4(m[k][4], m[k][5], m[k][6], m[k][7]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) sq += (double)u[k][e] * (double)u[k][e];
                }
            }
        }
    }
    for (int64_t i0 = done + start; i0 < count; i0 += 8 * step) {
        float u[8], m[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t i = i0 + k * step;
            u[k] = i < count ? ns_in(g[i]) : 0.0f;
            m[k] = mom && i < count ? mom[i] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t i = i0 + k * step;
            if (mom && i < count) {
                m[k] = fmaf(A.mu, m[k], u[k]);
                mom[i] = m[k];
                u[k] = A.nesterov ? fmaf(A.mu, m[k], u[k]) : m[k];
            }
            sq += (double)u[k] * (double)u[k];
        }
    }
    sq = ns_block_sum(sq, part);
    if (threadIdx.x == 0) J.parts[me] = sq;
}

// two values next to each other as their fp16 parts
__device__ __forceinline__ void ns_split(float v0, float v1, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(v0, v1);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(v0 - f.x, v1 - f.y);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// where the 16-byte chunk (8 columns from c on) of element (r, c) begins, in blocks of cbs column blocks per row block
__device__ __forceinline__ unsigned char *ns_chunk(unsigned char *x, int cbs, int r, int c)
{
    return x + ((int64_t)(r >> 7) * cbs + (c >> 6)) * (kParts * kBlock) + (r & 127) * 128 + (((c >> 3) & 7) ^ (r & 7)) * 16;
}

// X0, as blocks: a thread makes a chunk of eight columns
template <typename T>
__global__ void __launch_bounds__(256) ns_normalise_kernel(const __grid_constant__ NsArgs A)
{
    __shared__ double part[32];
    const NsJob &J = A.job[ns_find<0>(A, blockIdx.x)];
    const int me = blockIdx.x - J.first[0];
    const double sq = ns_block_sum((int)threadIdx.x < J.norm_parts ? J.parts[threadIdx.x] : 0.0, part);
    const NsScale scale(sq, A.eps);
    const T *g = (const T *)J.src;
    const bool tall = J.rows > J.cols, wide = !tall && J.cols % 8 == 0 && ns_wide(g) && ns_wide(J.mom);
    const int rows = ns_rb(J.m) * 128, cbs = ns_cb(J.n), chunks = cbs * 8;
    const unsigned total = (unsigned)rows * chunks;           // at most 2^28
    for (unsigned i = me * 256 + threadIdx.x; i < total; i += J.norm_parts * 256) {
        // neighbours in a warp read neighbours in memory: chunks of a row, or (tall) rows of a chunk
        const int r = tall ? (int)(i % (unsigned)rows) : (int)(i / (unsigned)chunks);
        const int c = (int)(tall ? i / (unsigned)rows : i % (unsigned)chunks) * 8;
        float v[8];
        if (wide && c < J.n) {
            if (r < J.m) {
                const int64_t at = (int64_t)r * J.cols + c;
                ns_load8(v, g + at);
                if (J.mom) {
                    float m[8];
                    ns_load8(m, J.mom + at);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = A.nesterov ? fmaf(A.mu, m[k], v[k]) : m[k];
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = r < J.m ? scale(v[k]) : 0.0f;
        } else
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = 0.0f;
            if (r < J.m && c + k < J.n) {
                const int64_t at = tall ? (int64_t)(c + k) * J.cols + r : (int64_t)r * J.cols + c + k;
                float u = ns_in(g[at]);
                if (J.mom) u = A.nesterov ? fmaf(A.mu, J.mom[at], u) : J.mom[at];
                v[k] = scale(u);
            }
        }
        uint4 hi, lo;
        ns_split(v[0], v[1], hi.x, lo.x);
        ns_split(v[2], v[3], hi.y, lo.y);
        ns_split(v[4], v[5], hi.z, lo.z);
        ns_split(v[6], v[7], hi.w, lo.w);
        unsigned char *at = ns_chunk(J.x[0], cbs, r, c);
        *(uint4 *)at = hi;
        *(uint4 *)(at + kBlock) = lo;
    }
}

// ------------------------------------------------------------------------------------------------ products
enum NsPhase { kGram, kPolynomial, kUpdate };

// MODE kAlone: a CTA makes tiles of 128 x 128.  kShared: so, and where there are few tiles several CTAs share one.  kPair: two CTAs
// make tiles of 256 x 256 together, each with half of either operand, so that a CTA loads as much per step for four times the
// products of a pair.
enum NsMode { kAlone, kShared, kPair };

template <int MODE>
struct NsTile {
    static constexpr int CG = MODE == kPair ? 2 : 1;
    static constexpr int TN = 128 * CG;                      // columns of the result, of which each CTA has 128 rows
    static constexpr int kA = kParts * kBlock, kB = kParts * kBlock, kStage = kA + kB;
    // a warp that loads, one that issues products, two to fill up; and those that take the results
    static constexpr int kTakers = 8, kThreads = 128 + 32 * kTakers;
    static constexpr int kWide = TN / (kTakers / 4), kPieces = kWide / 32;       // columns of a warp's 32 rows, pieces
    static constexpr int kPiece = 32 * 33 * 4;               // a 32 x 32 piece of each of these warps
    static constexpr int kExchange = MODE == kShared ? 128 * 128 * 4 : 0;          // the sums of those that share a tile
    static constexpr int kFixed = 1024 + 512 + kTakers * kPiece + kExchange;
    static constexpr int kStages = (227 * 1024 - kFixed) / kStage;
    static constexpr size_t kSmem = kFixed + (size_t)kStages * kStage;
    // Of `steps` steps of 64, how many have their sum in tensor memory at a time.  The tensor core cuts what it adds to a sum instead of
    // rounding it: over the 375 additions of a sum of 2000 products of two parts each that is a bias of 1e-5, ten times the rounding
    // of fp32 sums.  So the sums of 64 products are added up in registers, rounded, while the next ones are made:
    // 2000 x 333 is 2.4e-6 off after five steps (fp32 products: 2.5e-6), with sums of 128 4e-6.  In a pair's tiles, groups of more
    // steps let the products run further ahead while a tile's results are taken, and long sums are further off in fp32 too:
    // 4096 x 4096 3.70 / 3.47 / 3.36 / 3.35 ms and 1.0 / 1.2 / 1.6 / 1.9e-6 off with groups of 1 / 2 / 3 / 4 (fp32 products 4.8e-6), 700 x 700
    // 1.5 / 2.0e-6 with 2 / 3 (2.7e-6), 260 x 140 0.9 / 1.8 / 2.1e-6 with 1 / 2 / 3 (1.6e-6).  Results that are rounded to 8 bits (brief)
    // can do with sums of 1024 products, a bias of 1e-5: 6 x 1023 x 2049 768 -> 715 us, 4096 x 4096 3.54 -> 3.42 ms.
    static __device__ __forceinline__ int group(int steps, bool brief)
    {
        return brief ? 16 : MODE != kPair || steps < 8 ? 1 : steps < 16 ? 2 : 3;
    }
};

// 32 rows x 32 columns of a block in global memory and a warp's piece of shared memory: row by row 64 bytes, of which a lane
// moves 16, four lanes side by side; in the piece the 16-byte chunks are turned so that a lane can take its own row
// without two lanes meeting in a bank.
__device__ __forceinline__ int ns_piece_at(int row, int chunk) { return row * 64 + ((chunk ^ (row >> 1)) & 3) * 16; }

// (r0 is a multiple of 32: rows that lie eight apart have their chunks at the same places)
__device__ __forceinline__ uint4 *ns_piece_line(unsigned char *block, int r0, int c0, int lane)
{
    return (uint4 *)(block + ((r0 & 96) + (lane >> 2)) * 128 + ((((c0 >> 3) & 4) + (lane & 3)) ^ (lane >> 2)) * 16);
}

// What the result is made of besides the product: of b, a; of x', x.
struct NsOld {
    uint4 v[kParts][4];
    // requested early, put into the piece when it is wanted
    __device__ __forceinline__ void request(const NsJob &J, int kind, int from, int r0, int c, int lane)
    {
        if (kind == kGram) return;
        const int cbs = kind == kUpdate ? ns_cb(J.n) : ns_cb(J.m);
        unsigned char *block = (kind == kPolynomial ? J.a : J.x[from]) + ((int64_t)(r0 >> 7) * cbs + (c >> 6)) * (kParts * kBlock);
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[p][i] = __ldcg(ns_piece_line(block, r0, c, lane) + (p * kBlock + i * 1024) / 16);
    }
    __device__ __forceinline__ void put(unsigned char *piece, int lane) const
    {
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) *(uint4 *)(piece + ns_piece_at(lane >> 2, lane & 3) + p * 2048 + i * 512) = v[p][i];
    }
};

// What a warp does with 32 rows (from r0, lane = row) x 32 columns (from c) of a result.  next: the columns of the piece that
// follows, whose old values are requested meanwhile, or -1.
template <typename T>
__device__ __forceinline__ void ns_take_piece(const NsArgs &A, const NsJob &J, int kind, bool last, int from, int r0, int c, float (&v)[32],
                                              unsigned char *piece, int lane, NsOld &old, int next)
{
    if (kind == kGram) {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] *= kScaleA / (kScaleX * kScaleX);
    } else {
        // b = cb a + ..., x' = ca x + ...
        const float f = kind == kPolynomial ? A.cb : A.ca, by = kind == kPolynomial ? A.cc / kScaleA : 1.0f / kScaleA;
        __syncwarp();
        old.put(piece, lane);
        __syncwarp();
        if (next >= 0) old.request(J, kind, from, r0, next, lane);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint4 hi = *(const uint4 *)(piece + ns_piece_at(lane, k));
            uint4 lo = make_uint4(0, 0, 0, 0);
            lo = *(const uint4 *)(piece + 2048 + ns_piece_at(lane, k));
            const uint32_t hs[4] = {hi.x, hi.y, hi.z, hi.w}, ls[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float2 o = __half22float2(*reinterpret_cast<const __half2 *>(&hs[e]));
                const float2 l = __half22float2(*reinterpret_cast<const __half2 *>(&ls[e]));
                o.x += l.x;
                o.y += l.y;
                v[8 * k + 2 * e] = fmaf(f, o.x, by * v[8 * k + 2 * e]);
                v[8 * k + 2 * e + 1] = fmaf(f, o.y, by * v[8 * k + 2 * e + 1]);
            }
        }
    }
    __syncwarp();
    if (last) {
        // to the weight, of which the piece is 32 x 32 as well, turned if it is tall: 16 bytes a lane where its rows allow it, else
        // 32 elements next to each other at a time
        constexpr int E = 16 / sizeof(T), U = 4;
        T *dst = (T *)J.dst;
        const bool tall = J.rows > J.cols, update = J.mom != nullptr;
        const int row0 = tall ? c : r0, col0 = tall ? r0 : c, rows = min(32, J.rows - row0), cols = min(32, J.cols - col0);
        const int64_t step = J.cols;
        const float keep = J.keep, by = update ? -J.step * (1.0f / kScaleX) : 1.0f / kScaleX;
        float *turned = (float *)piece;
#pragma unroll
        for (int k = 0; k < 32; ++k) turned[tall ? k * 33 + lane : lane * 33 + k] = v[k];
        __syncwarp();
        if (J.cols % E == 0 && ns_wide(dst)) {
            const int row = lane / (32 / E), col = lane % (32 / E) * E;
            const float *from = turned + row * 33 + col;
            T *at = dst + (row0 + row) * step + col0 + col;
#pragma unroll
            for (int i0 = 0; i0 < 32 / E; i0 += U) {
                uint4 w[U];
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (update && row + (i0 + i) * E < rows && col < cols) w[i] = *(const uint4 *)(at + (i0 + i) * E * step);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float o[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = from[(i0 + i) * E * 33 + e] * by;
                    if (row + (i0 + i) * E < rows && col < cols) ns_store16<T>(at + (i0 + i) * E * step, o, w[i], keep, update);
                }
            }
        } else {
            T *at = dst + row0 * step + col0 + lane;
#pragma unroll 1
            for (int k0 = 0; k0 < rows; k0 += 8) {
                float w[8], o[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = update && lane < cols && k0 + k < rows ? ns_in(at[k * step]) : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = turned[(k0 + k) * 33 + lane] * by;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (lane < cols && k0 + k < rows) at[k * step] = ns_out<T>(update ? fmaf(keep, w[k], o[k]) : o[k]);
                at += 8 * step;
            }
        }
        __syncwarp();
    } else {
        const int cbs = kind == kUpdate ? ns_cb(J.n) : ns_cb(J.m);
        unsigned char *to = (kind == kGram ? J.a : kind == kPolynomial ? J.b : J.x[from ^ 1]) + ((int64_t)(r0 >> 7) * cbs + (c >> 6)) * (kParts * kBlock);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint4 hi, lo;
            ns_split(v[8 * k], v[8 * k + 1], hi.x, lo.x);
            ns_split(v[8 * k + 2], v[8 * k + 3], hi.y, lo.y);
            ns_split(v[8 * k + 4], v[8 * k + 5], hi.z, lo.z);
            ns_split(v[8 * k + 6], v[8 * k + 7], hi.w, lo.w);
            *(uint4 *)(piece + ns_piece_at(lane, k)) = hi;
            *(uint4 *)(piece + 2048 + ns_piece_at(lane, k)) = lo;
        }
        __syncwarp();
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                ns_piece_line(to, r0, c, lane)[(p * kBlock + i * 1024) / 16] = *(const uint4 *)(piece + ns_piece_at(lane >> 2, lane & 3) + p * 2048 + i * 512);
    }
}

// All steps in one launch: three phases each,
//   kGram        a = x x^T
//   kPolynomial  b = cb a + cc a a
//   kUpdate      x' = ca x + b x; in the last step the result goes to the weight
// with all CTAs resident (a cooperative launch) and waiting for one another between phases: the small matrices' products take a
// few microseconds, as long as a launch and the way of its first loads.  In a phase a CTA (a pair of them) takes tiles of the result.
// a and b are symmetric: their blocks below the diagonal are neither computed nor stored.  Where a product wants one as
// rows, it takes the block across the diagonal as columns.
//
// In mode kShared split[phase] CTAs of a cluster share a tile: each sums over its part of the steps of the summation
// index, they exchange the sums through shared memory, and each takes some 32 x 32 pieces of the total, added up in the order
// of the ranks.
struct NsPlan {
    int steps;
    int tiles[3], split[3];          // by phase
    unsigned *arrived;               // zero before the launch
    int *status;
};

template <int MODE, typename T>
__global__ void __launch_bounds__(NsTile<MODE>::kThreads, 1) ns_steps_kernel(const __grid_constant__ NsArgs A, const __grid_constant__ NsPlan P)
{
    using Tile = NsTile<MODE>;
    constexpr int CG = Tile::CG, S = Tile::kStages, TN = Tile::TN, kTakers = Tile::kTakers, kPieces = Tile::kPieces;
    // pieces of the old values that a warp requests before its sums are complete (as many as the registers hold)
    constexpr int kAhead = MODE != kAlone ? 1 : kPieces;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    // full: this CTA's loads are there; ready: the second CTA's are (at the first); empty: a stage has been read; done: a sum is
    // complete; taken: it has been taken out; given: the sums of all that share a tile are there
    uint64_t *full = (uint64_t *)(smem + S * Tile::kStage), *ready = full + S, *empty = ready + S, *done = empty + S, *taken = done + 2;
    uint64_t *given = taken + 2;
    uint32_t *base_at = (uint32_t *)(given + 3);
    unsigned char *pieces = smem + S * Tile::kStage + 512, *exchange = pieces + kTakers * Tile::kPiece;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = CG == 2 ? rank : 0;
    const bool clustered = cluster_size() > 1;
    if (warp == 1) tensor_alloc<CG>(base_at, 2 * TN);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(full + i, 1);
            mbar_init(ready + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(done + i, 1);
            mbar_init(taken + i, kTakers * CG);
        }
        for (int i = 0; i < 3; ++i) mbar_init(given + i, kTakers * P.split[i]);
        mbar_init_fence();
    }
    tensor_fence_before();
    __syncthreads();
    if (clustered) cluster_wait_all();
    tensor_fence_after();
    const uint32_t acc = *base_at;
    bool fine = true;

    // a phase: which tiles this CTA takes, and its part of the summation index
    struct Phase {
        int kind, from, tile, step, tiles, split, rank;
        bool last;
    };
    auto phase_of = [&](int ph) {
        Phase p;
        p.kind = ph % 3;
        p.from = ph / 3 & 1;
        p.last = ph + 1 == 3 * P.steps;
        p.tiles = P.tiles[p.kind];
        p.split = P.split[p.kind];
        const int width = CG == 2 ? 2 : p.split;
        p.tile = blockIdx.x / width;
        p.step = gridDim.x / width;
        p.rank = rank % p.split;
        return p;
    };
    // tile -> its job, its first row block and its first column block, and this CTA's part of the summation index
    struct Spot {
        int job, i, j, k0, k1;
    };
    auto locate = [&](const Phase &p, int tile) {
        Spot o;
        const bool symmetric = p.kind != kUpdate;
        int n = 0;
        while (n + 1 < A.jobs && A.job[n + 1].first[symmetric ? 1 : 2] <= tile) ++n;
        o.job = n;
        const NsJob &J = A.job[n];
        int at = tile - J.first[symmetric ? 1 : 2];
        const int rt = (ns_rb(J.m) + CG - 1) / CG;
        if (symmetric) {
            // a row of tiles begins at the diagonal
            for (o.i = 0; at >= rt - o.i; ++o.i) at -= rt - o.i;
            o.j = o.i + at;
        } else {
            // tiles that run side by side share columns of x
            o.i = at % rt;
            o.j = at / rt;
        }
        o.i *= CG;
        o.j *= CG;
        const int steps = p.kind == kGram ? ns_cb(J.n) : ns_cb(J.m);
        o.k0 = steps * p.rank / p.split;
        o.k1 = steps * (p.rank + 1) / p.split;
        return o;
    };
    // The same tiles in every step: the first few are worked out once (some 300 instructions one after the other, which would stand
    // between the phases, and between the tiles of a phase).
    constexpr int kSpots = 4;
    __shared__ Phase phases[3];
    __shared__ Spot spots[3][kSpots];
    if (threadIdx.x < 3 * kSpots) {
        const int kind = threadIdx.x / kSpots, it = threadIdx.x % kSpots;
        const Phase p = phase_of(kind);
        if (it == 0) phases[kind] = p;
        if (p.tile + it * p.step < p.tiles) spots[kind][it] = locate(p, p.tile + it * p.step);
    }
    __syncthreads();
    auto phase_at = [&](int ph, int kind) {
        Phase p = phases[kind];
        p.from = ph / 3 & 1;
        p.last = ph + 1 == 3 * P.steps;
        return p;
    };
    auto spot_at = [&](const Phase &p, int tile, int it) { return it < kSpots ? spots[p.kind][it] : locate(p, tile); };
    // whether step k takes an operand from across the diagonal (of the two row blocks of a pair, which take it alike, one may be the
    // diagonal's own, which is the same either way)
    auto left_turned = [&](int kind, int i, int k) { return kind != kGram && (k >> 1) < i + CG - 1; };
    auto right_turned = [&](int kind, int j, int k) { return kind == kPolynomial ? (k >> 1) < j + CG - 1 : kind == kUpdate; };

    if (warp < 4) {
        // 128 threads give registers to the 256 that hold sums: 128 * 40 + 256 * 224 = 128 * 56 + 256 * 216 <= 384 * 168.  (A pair's sums
        // of 128 columns need the last eight; elsewhere the loads' addresses do.)
        if constexpr (MODE == kPair) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 && lane == 0) {
            int s = 0, turn = 0;
            for (int ph = 0, kind = 0; fine && ph < 3 * P.steps; ++ph, kind = kind == 2 ? 0 : kind + 1) {
                if (ph > 0) {
                    if (!grid_wait_bounded(P.arrived, ph * gridDim.x, kWaitLimit)) { fine = false; break; }
                    fence_async_global();
                }
                const Phase p = phase_at(ph, kind);
                for (int tile = p.tile, it = 0; fine && tile < p.tiles; tile += p.step, ++it) {
                    const Spot o = spot_at(p, tile, it);
                    const NsJob &J = A.job[o.job];
                    const int cbm = ns_cb(J.m), cbn = ns_cb(J.n), rb = ns_rb(J.m);
                    const int cbl = p.kind == kGram ? cbn : cbm, cbr = p.kind == kPolynomial ? cbm : cbn;
                    const unsigned char *left = p.kind == kGram ? J.x[p.from] : p.kind == kPolynomial ? J.a : J.b;
                    const unsigned char *right = p.kind == kPolynomial ? J.a : J.x[p.from];
                    const int il = o.i + pair, jr = o.j + pair;        // this CTA's row block and column block; behind the last one, nothing
                    const bool has_left = il < rb, has_right = jr < (p.kind != kUpdate ? rb : ns_rb(J.n));
                    const unsigned bytes = kParts * kBlock * (has_left + has_right);
                    // 64 rows of two blocks of 64 columns: [part][column block]
                    auto columns = [&](unsigned char *to, const unsigned char *x, int cbs, int k, int block) {
                        const unsigned char *row = x + ((int64_t)(k >> 1) * cbs + 2 * block) * (kParts * kBlock) + (k & 1) * (kBlock / 2);
                        for (int b = 0; b < 2; ++b)
                            for (int q = 0; q < kParts; ++q)
                                bulk_load(to + q * kBlock + b * (kBlock / 2), row + (b * kParts + q) * kBlock, kBlock / 2, full + s);
                    };
                    for (int k = o.k0; k < o.k1; ++k) {
                        if (!mbar_wait_bounded(empty + s, turn ^ 1, kWaitLimit)) { fine = false; break; }
                        unsigned char *to = smem + s * Tile::kStage;
                        mbar_expect_tx(full + s, bytes);
                        if (has_left) {
                            if (left_turned(p.kind, o.i, k)) columns(to, left, cbl, k, il);
                            else bulk_load(to, left + ((int64_t)il * cbl + k) * (kParts * kBlock), kParts * kBlock, full + s);
                        }
                        to += Tile::kA;
                        if (has_right) {
                            if (right_turned(p.kind, o.j, k)) columns(to, right, cbr, k, jr);
                            else bulk_load(to, right + ((int64_t)jr * cbr + k) * (kParts * kBlock), kParts * kBlock, full + s);
                        }
                        if (++s == S) { s = 0; turn ^= 1; }
                    }
                }
            }
            // every stage's last copy has been read before the CTA leaves
            for (int k = 0; k < S; ++k) {
                if (!mbar_wait_bounded(empty + s, turn ^ 1, kWaitLimit)) fine = false;
                if (++s == S) { s = 0; turn ^= 1; }
            }
        } else if (warp == 1 && lane == 0 && pair == 0) {
            int s = 0, turn = 0, slot = 0, again = 0;
            for (int ph = 0, kind = 0; fine && ph < 3 * P.steps; ++ph, kind = kind == 2 ? 0 : kind + 1) {
                const Phase p = phase_at(ph, kind);
                for (int tile = p.tile, it = 0; fine && tile < p.tiles; tile += p.step, ++it) {
                    const Spot o = spot_at(p, tile, it);
                    const int group = Tile::group(o.k1 - o.k0, std::is_same<T, __nv_bfloat16>::value);
                    for (int k = o.k0, in = 0; k < o.k1; ++k) {
                        const bool first = in == 0;
                        if (first && !mbar_wait_bounded(taken + slot, again ^ 1, kWaitLimit)) { fine = false; break; }
                        if (!mbar_wait_bounded(full + s, turn, kWaitLimit)) { fine = false; break; }
                        if (CG == 2 && !mbar_wait_bounded(ready + s, turn, kWaitLimit)) { fine = false; break; }
                        tensor_fence_after();
                        const unsigned a0 = smem_u32(smem + s * Tile::kStage), b0 = a0 + Tile::kA;
                        const bool lt = left_turned(p.kind, o.i, k), rt = right_turned(p.kind, o.j, k);
                        const uint32_t shape = product_shape(128 * CG, TN, lt, rt), d = acc + slot * TN;
                        // descriptors count 16 bytes: 16 columns are 2 further, 16 rows 128, the other part a block
                        const uint64_t l = lt ? desc_columns(a0, kBlock / 2) : desc_rows(a0), r = rt ? desc_columns(b0, kBlock / 2) : desc_rows(b0);
                        const unsigned dl = lt ? 128 : 2, dr = rt ? 128 : 2, other = kBlock / 16;
                        // the small products first: what they lose to the sum's size is less while it is small
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            product<CG>(d, l + q * dl, r + q * dr + other, shape, !first || q > 0);
                            product<CG>(d, l + q * dl + other, r + q * dr, shape, true);
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) product<CG>(d, l + q * dl, r + q * dr, shape, true);
                        product_commit<CG>(empty + s);
                        if (++s == S) { s = 0; turn ^= 1; }
                        if (++in == group || k + 1 == o.k1) {
                            in = 0;
                            product_commit<CG>(done + slot);
                            if ((slot ^= 1) == 0) again ^= 1;
                        }
                    }
                }
            }
        } else if (CG == 2 && warp == 1 && lane == 0) {
            // the second CTA tells the first what it has loaded
            int s = 0, turn = 0;
            for (int ph = 0, kind = 0; fine && ph < 3 * P.steps; ++ph, kind = kind == 2 ? 0 : kind + 1) {
                const Phase p = phase_at(ph, kind);
                for (int tile = p.tile, it = 0; fine && tile < p.tiles; tile += p.step, ++it) {
                    const Spot o = spot_at(p, tile, it);
                    for (int k = o.k0; k < o.k1; ++k) {
                        if (!mbar_wait_bounded(full + s, turn, kWaitLimit)) { fine = false; break; }
                        mbar_arrive_at(ready + s, 0);
                        if (++s == S) { s = 0; turn ^= 1; }
                    }
                }
            }
        }
        __syncwarp();
    } else {
        if constexpr (MODE == kPair) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        int slot = 0, again = 0;
        const int w = warp - 4, quarter = warp & 3;
        unsigned char *piece = pieces + w * Tile::kPiece;
        for (int ph = 0, kind = 0; fine && ph < 3 * P.steps; ++ph, kind = kind == 2 ? 0 : kind + 1) {
            const Phase p = phase_at(ph, kind);
            // what the phase before has left, for what is requested before the products are done; and a CTA without a tile must not
            // arrive before its time
            if (ph > 0) {
                if (lane == 0) fine = grid_wait_bounded(P.arrived, ph * gridDim.x, kWaitLimit);
                fine = __all_sync(0xffffffffu, fine);
            }
            for (int tile = p.tile, it = 0; fine && tile < p.tiles; tile += p.step, ++it) {
                const Spot o = spot_at(p, tile, it);
                const NsJob &J = A.job[o.job];
                const int group = Tile::group(o.k1 - o.k0, std::is_same<T, __nv_bfloat16>::value), groups = (o.k1 - o.k0 + group - 1) / group, rb = ns_rb(J.m);
                const int il = o.i + pair, c0 = (w >> 2) * Tile::kWide, jl = o.j + (c0 >> 7);      // this warp's columns of the tile; its blocks
                const bool mine = il < rb && jl < (p.kind != kUpdate ? rb : ns_rb(J.n)) && !(p.kind != kUpdate && jl < il);
                const int r0 = il * 128 + quarter * 32, c = o.j * 128 + c0;
                const uint32_t at = acc + ((uint32_t)(quarter * 32) << 16) + c0;
                float sum[kPieces][32];
#pragma unroll
                for (int u = 0; u < kPieces; ++u)
#pragma unroll
                    for (int k = 0; k < 32; ++k) sum[u][k] = 0.0f;
                NsOld old[kAhead];
                if (mine && !(MODE == kShared && p.split > 1)) {
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) old[u].request(J, p.kind, p.from, r0, c + u * 32, lane);
                }
                // To the one of those that share the tile whose piece it is: pieces rank, rank + split, ... of the sixteen, from every
                // rank in turn.  (Written there, not fetched: a read of another CTA's memory takes 400 cycles, and the stores are
                // on their way together.)
                auto give = [&](const float (&v)[32], int u) {
                    const int id = ((c0 >> 5) + u) * 4 + quarter, to = id & (p.split - 1);
                    float4 *at = (float4 *)exchange + (p.rank * (16 / p.split) + id / p.split) * 256 + lane;
#pragma unroll
                    for (int k = 0; k < 8; ++k) write_at(at + k * 32, rank - p.rank + to, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
                };
                auto pass_on = [&](float (&v)[32], int u) {
                    if (MODE == kShared && p.split > 1) {
                        give(v, u);
                    } else {
                        ns_take_piece<T>(A, J, p.kind, p.last, p.from, r0, c + u * 32, v, piece, lane, old[u % kAhead], u + kAhead < kPieces ? c + (u + kAhead) * 32 : -1);
                    }
                };
                for (int g = 0; g < groups; ++g) {
                    if (!__all_sync(0xffffffffu, mbar_wait_bounded(done + slot, again, kWaitLimit))) { fine = false; break; }
                    tensor_fence_after();
                    if (mine) {
#pragma unroll
                        for (int u = 0; u < kPieces; ++u) {
                            float v[32];
                            tensor_read(v, at + slot * TN + u * 32);
#pragma unroll
                            for (int k = 0; k < 32; ++k) sum[u][k] += v[k];
                        }
                    }
                    tensor_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) mbar_arrive_at(taken + slot, 0);
                        else mbar_arrive(taken + slot);
                    }
                    if ((slot ^= 1) == 0) again ^= 1;
                }
                if (MODE == kShared && p.split > 1) {
#pragma unroll
                    for (int u = 0; u < kPieces; ++u) give(sum[u], u);
                } else if (fine && mine) {
#pragma unroll
                    for (int u = 0; u < kPieces; ++u) {
                        pass_on(sum[u], u);
                    }
                }
            }
            if (MODE == kShared && p.split > 1) {
                __syncwarp();
                if (lane < p.split) mbar_release_at(given + p.kind, rank - p.rank + lane);
                if (p.tile < p.tiles) {
                    const Spot &o = spots[kind][0];
                    // this CTA's pieces of 32 x 32; warp w takes the w-th of them
                    const int many = 16 / p.split, id = w * p.split + p.rank, part = id & 3, c = id >> 2;
                    NsOld old;
                    if (w < many) old.request(A.job[o.job], p.kind, p.from, o.i * 128 + part * 32, o.j * 128 + c * 32, lane);
                    fine = __all_sync(0xffffffffu, mbar_acquire_bounded(given + p.kind, ph / 3 & 1, kWaitLimit)) && fine;
                    if (w < many) {
                        float v[32] = {};
                        for (int r = 0; r < p.split; ++r) {
                            const float4 *at = (const float4 *)exchange + (r * many + w) * 256 + lane;
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float4 x = at[k * 32];
                                v[4 * k] += x.x;
                                v[4 * k + 1] += x.y;
                                v[4 * k + 2] += x.z;
                                v[4 * k + 3] += x.w;
                            }
                        }
                        ns_take_piece<T>(A, A.job[o.job], p.kind, p.last, p.from, o.i * 128 + part * 32, o.j * 128 + c * 32, v, piece, lane, old, -1);
                    }
                }
            }
            if (!p.last) {
                // what this CTA has written is there for the others' loads
                if (MODE == kShared && p.split > 1) fence_async_all();
                else fence_async_global();
                fine = all_agree(1, 32 * kTakers, fine);   // a warp that gave up takes the others along
                if (threadIdx.x == 128) grid_arrive(P.arrived);
            }
        }
        __syncwarp();
    }
    if (!fine) atomicExch(P.status, kStatusNsTimeout);
    tensor_fence_before();
    __syncthreads();
    if (clustered) cluster_wait_all();               // no CTA leaves while another reads its memory or arrives at its barriers
    if (warp == 1) {
        tensor_fence_after();
        tensor_free<CG>(acc, 2 * TN);
    }
}

// ------------------------------------------------------------------------------------------- small matrices
// Up to 128 rows: a matrix stays in the shared memory of a cluster from its gradient to its weight's update, in one launch.  Each
// CTA has some column blocks of 64 of X and all of A.  A step: every CTA's part of X X^T, added up across the cluster (each CTA
// adds up its share and gives it to all); A A by every CTA for itself; B X of its own columns, in place.  What bounds it is latency:
// a step is three products of a microsecond and the way through tensor memory, registers and shared memory between them.
// A block here has only as many rows as the matrix (a multiple of 16); the tensor core reads 128, and what lies behind gives
// rows of the result that nobody looks at.
constexpr int kSmallThreads = 512;
constexpr int kSmallScratch = 16 * 32 * 17 * 4;          // a 32 x 16 piece of each warp

struct NsSmall {
    int rows, per, block, x, ab, scratch, sums, spread, total;         // rows and bytes
    bool fits, few;
};

// where things lie in the shared memory of a CTA with `per` column blocks of a matrix of m rows
static __host__ __device__ __forceinline__ NsSmall ns_small(int m, int per)
{
    NsSmall s;
    s.rows = (m + 15) / 16 * 16;
    s.per = per;
    s.block = kParts * s.rows * 128;
    s.x = per * s.block;
    // A, later B: as blocks; before that, fp32 sums for the exchange.  The last operand's 128 rows reach 16 KB behind its start.
    const int abs = (s.rows + 63) / 64 * s.block, sums = s.rows * s.rows * 4, reach = abs - s.rows * 128 + kBlock;
    s.ab = abs > sums ? abs : sums;
    s.ab = s.ab > reach ? s.ab : reach;
    // results on their way to the weight: over B where all columns fit tensor memory at once, so that B is not needed any more
    s.scratch = s.rows > 64 ? s.x : s.x + s.ab;
    s.total = s.rows > 64 ? s.x + (s.ab > kSmallScratch ? s.ab : kSmallScratch) : s.scratch + kSmallScratch;
    // of up to 32 rows, all CTAs' sums (of two steps), and a product on its way to threads that cannot read its tensor memory
    s.few = s.rows <= 32 && per <= 8 && s.total + 2 * 8 * sums + per * 64 * s.rows * 4 <= 226 * 1024 - 1024;
    s.sums = s.total;
    s.spread = s.sums + 2 * 8 * sums;
    if (s.few) s.total = s.spread + per * 64 * s.rows * 4;
    s.fits = s.total <= 226 * 1024 - 1024 && (s.rows <= 64 || per <= 8);
    return s;
}

// u of eight columns from c on of row r (0 outside the matrix); first: the momentum is brought up to date on the way
template <typename T>
__device__ __forceinline__ void ns_load_u(const NsArgs &A, const NsJob &J, int r, int c, bool first, float (&v)[8])
{
    const T *g = (const T *)J.src;
    const bool tall = J.rows > J.cols, wide = !tall && J.cols % 8 == 0 && ns_wide(g) && ns_wide(J.mom);
    const int64_t at0 = tall ? (int64_t)c * J.cols + r : (int64_t)r * J.cols + c, step = tall ? J.cols : 1;
    float m[8];
    if (wide) {
        if (c < J.n) {
            ns_load8(v, g + at0);
            if (J.mom) ns_load8(m, J.mom + at0);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = m[k] = 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = c + k < J.n ? ns_in(g[at0 + k * step]) : 0.0f;
            m[k] = J.mom && c + k < J.n ? J.mom[at0 + k * step] : 0.0f;
        }
    }
    if (J.mom) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (first) {
                m[k] = fmaf(A.mu, m[k], v[k]);
                if (c + k < J.n) J.mom[at0 + k * step] = m[k];
            }
            v[k] = A.nesterov ? fmaf(A.mu, m[k], v[k]) : m[k];
        }
    }
}

// sixteen columns of a row, as two chunks of a block
__device__ __forceinline__ void ns_put16(unsigned char *row, int part_bytes, int chunk, int r, const float (&v)[16])
{
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint4 hi, lo;
        ns_split(v[8 * k], v[8 * k + 1], hi.x, lo.x);
        ns_split(v[8 * k + 2], v[8 * k + 3], hi.y, lo.y);
        ns_split(v[8 * k + 4], v[8 * k + 5], hi.z, lo.z);
        ns_split(v[8 * k + 6], v[8 * k + 7], hi.w, lo.w);
        unsigned char *at = row + (((chunk + k) ^ r) & 7) * 16;
        *(uint4 *)at = hi;
        *(uint4 *)(at + part_bytes) = lo;
    }
}

// v <- f old + by v for the same
__device__ __forceinline__ void ns_add16(const unsigned char *row, int part_bytes, int chunk, int r, float f, float by, float (&v)[16])
{
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const unsigned char *at = row + (((chunk + k) ^ r) & 7) * 16;
        const uint4 hi = *(const uint4 *)at;
        uint4 lo = make_uint4(0, 0, 0, 0);
        lo = *(const uint4 *)(at + part_bytes);
        const uint32_t hs[4] = {hi.x, hi.y, hi.z, hi.w}, ls[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 o = __half22float2(*reinterpret_cast<const __half2 *>(&hs[e]));
            const float2 l = __half22float2(*reinterpret_cast<const __half2 *>(&ls[e]));
            o.x += l.x;
            o.y += l.y;
            v[8 * k + 2 * e] = fmaf(f, o.x, by * v[8 * k + 2 * e]);
            v[8 * k + 2 * e + 1] = fmaf(f, o.y, by * v[8 * k + 2 * e + 1]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kSmallThreads, 1) ns_small_kernel(const __grid_constant__ NsArgs A, int steps, int *status)
{
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t bar;
    __shared__ uint32_t base_at;
    __shared__ double part[32], square;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = (int)cluster_size(), rank = (int)cluster_rank();
    const NsJob &J = A.job[blockIdx.x / C];
    const int blocks = (J.n + 63) / 64;
    const NsSmall L = ns_small(J.m, (blocks + C - 1) / C);
    const int b0 = min(rank * L.per, blocks), nb = min(L.per, blocks - b0), R = L.rows, side = R * 128;
    unsigned char *x = smem, *ab = smem + L.x;
    if (warp == 0) tensor_alloc<1>(&base_at, 512);
    if (tid == 0) {
        mbar_init(&bar, 1);
        mbar_init_fence();
    }

    // momentum and norm
    const int chunks = nb * 8;
    const bool tall = J.rows > J.cols;
    double sq = 0.0;
    for (int i = tid; i < J.m * chunks; i += kSmallThreads) {
        float v[8];
        ns_load_u<T>(A, J, tall ? i % J.m : i / chunks, b0 * 64 + (tall ? i / J.m : i % chunks) * 8, true, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) sq += (double)v[k] * (double)v[k];
    }
    sq = ns_block_sum(sq, part);
    if (tid == 0) square = sq;
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t acc = base_at;
    if (C > 1) {
        cluster_wait_all();
        sq = 0.0;
        for (int r = 0; r < C; ++r) sq += read_double_at(&square, r);
    }
    const NsScale scale(sq, A.eps);
    for (int i = tid; i < R * chunks; i += kSmallThreads) {
        const int r = tall ? i % R : i / chunks, ch = tall ? i / R : i % chunks;
        float v[8] = {};
        if (r < J.m) ns_load_u<T>(A, J, r, b0 * 64 + ch * 8, false, v);
        uint4 hi, lo;
        ns_split(scale(v[0]), scale(v[1]), hi.x, lo.x);
        ns_split(scale(v[2]), scale(v[3]), hi.y, lo.y);
        ns_split(scale(v[4]), scale(v[5]), hi.z, lo.z);
        ns_split(scale(v[6]), scale(v[7]), hi.w, lo.w);
        unsigned char *at = x + (ch >> 3) * L.block + r * 128 + ((ch ^ r) & 7) * 16;
        *(uint4 *)at = hi;
        *(uint4 *)(at + side) = lo;
    }

    // this warp's rows of a result, and its first sixteen columns of each 64
    const int r = (warp & 3) * 32 + lane, first = (warp >> 2) * 16;
    const bool mine = (warp & 3) * 32 < R, row_there = r < R;
    const uint32_t at = acc + ((uint32_t)((warp & 3) * 32) << 16);
    bool fine = true;
    int turn = 0;
    // what has been written to shared memory is there for the products; what is in tensor memory has been read
    const auto ready = [&] {
        fence_proxy_async();
        tensor_fence_before();
        __syncthreads();
        tensor_fence_after();
    };
    const auto made = [&] {
        if (!mbar_wait_bounded(&bar, turn, kWaitLimit)) fine = false;
        turn ^= 1;
        __syncwarp();
        tensor_fence_after();
    };
    const unsigned xs = smem_u32(x), abs = smem_u32(ab);
    // up to four steps of 16 of the summation index, descriptors dl and dr apart: the small products first, what they lose to the
    // sum's size is less while it is small
    const unsigned other = side / 16;
    const auto multiply = [&](uint32_t d, uint64_t left, unsigned dl, uint64_t right, unsigned dr, uint32_t shape, int count, bool add) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < count) {
                product<1>(d, left + q * dl, right + q * dr + other, shape, add || q > 0);
                product<1>(d, left + q * dl + other, right + q * dr, shape, true);
            }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < count) product<1>(d, left + q * dl, right + q * dr, shape, true);
    };
    // sums of a few blocks each, added up in registers (see NsTile::group); those of A A and B X have 64 products each too, where tensor
    // memory has room (with sums of 128: 128 x 1024 119.5 us instead of 121.2, and 3.9e-6 off instead of 2.4e-6)
    const int sums = max(1, min(512 / R, (nb + 1) / 2));

    for (int s = 0; s < steps; ++s) {
        const bool last = s + 1 == steps;
        ready();
        if (tid == 0) {
            for (int g = 0; g < sums; ++g)
                for (int b = nb * g / sums; b < nb * (g + 1) / sums; ++b) {
                    const uint64_t rows = desc_rows(xs + b * L.block);
                    multiply(acc + g * R, rows, 2, rows, 2, product_shape(128, R, false, false), 4, b > nb * g / sums);
                }
            product_commit<1>(&bar);
        }
        made();
        if (mine)
            for (int c = first; c < R; c += 64) {
                float v[16], t[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = 0.0f;
                __syncwarp();
                if (nb > 0)
                    for (int g = 0; g < sums; ++g) {
                        tensor_read(t, at + g * R + c);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] += t[k];
                    }
                if (row_there && C == 1) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] *= kScaleA / (kScaleX * kScaleX);
                    ns_put16(ab + (c >> 6) * L.block + r * 128, side, (c >> 3) & 7, r, v);
                } else if (row_there) {
                    // four columns of all rows after one another; few rows, to everybody
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float4 sum = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                        const int e = (c / 4 + k) * R + r;
                        if (L.few)
                            for (int o = 0; o < C; ++o) write_at((float4 *)(smem + L.sums) + ((s & 1) * 8 + rank) * (R * R / 4) + e, o, sum);
                        else ((float4 *)ab)[e] = sum;
                    }
                }
            }
        if (C > 1 && L.few) {
            // (a CTA that is a step ahead writes to the other half)
            __syncwarp();
            cluster_wait_all();
            const float4 *sums = (const float4 *)(smem + L.sums) + (s & 1) * 8 * (R * R / 4);
            if (tid < R * R / 4) {
                float4 total = sums[tid];
                for (int o = 1; o < C; ++o) {
                    const float4 y = sums[o * (R * R / 4) + tid];
                    total.x += y.x;
                    total.y += y.y;
                    total.z += y.z;
                    total.w += y.w;
                }
                const float f = kScaleA / (kScaleX * kScaleX);
                const int row = tid % R, c = tid / R * 4;
                uint2 hi, lo;
                ns_split(total.x * f, total.y * f, hi.x, lo.x);
                ns_split(total.z * f, total.w * f, hi.y, lo.y);
                unsigned char *to = ab + row * 128 + ((((c >> 3) ^ row) & 7) * 16) + (c & 4) * 2;
                *(uint2 *)to = hi;
                *(uint2 *)(to + side) = lo;
            }
        } else if (C > 1) {
            __syncwarp();
            cluster_wait_all();
            const int all = R * R / 4, e0 = all * rank / C, e1 = all * (rank + 1) / C;
            float4 total[4];                             // 128 * 128 / 4 / 2 / 512
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = e0 + tid + k * kSmallThreads;
                total[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (e < e1) {
                    float4 y[8];
#pragma unroll
                    for (int o = 0; o < 8; ++o)
                        if (o < C) y[o] = read_at((const float4 *)ab + e, o);
#pragma unroll
                    for (int o = 0; o < 8; ++o)
                        if (o < C) {
                            total[k].x += y[o].x;
                            total[k].y += y[o].y;
                            total[k].z += y[o].z;
                            total[k].w += y[o].w;
                        }
                }
            }
            __syncwarp();
            cluster_wait_all();                          // all sums have been read: A takes their place
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = e0 + tid + k * kSmallThreads, row = e % R, c = e / R * 4;
                if (e < e1) {
                    const float f = kScaleA / (kScaleX * kScaleX);
                    uint32_t h0, h1, l0, l1;
                    ns_split(total[k].x * f, total[k].y * f, h0, l0);
                    ns_split(total[k].z * f, total[k].w * f, h1, l1);
                    unsigned char *to = ab + (c >> 6) * L.block + row * 128 + ((((c >> 3) ^ row) & 7) * 16) + (c & 4) * 2;
                    for (int o = 0; o < C; ++o) {
                        write_at(to, o, h0, h1);
                        write_at(to + side, o, l0, l1);
                    }
                }
            }
            fence_async_all();
            __syncwarp();
            cluster_wait_all();
        }
        ready();
        if (tid == 0) {
            for (int k = 0; k < R; k += 64) {
                const uint64_t rows = desc_rows(abs + (k >> 6) * L.block);
                multiply(acc + (k >> 6) * R, rows, 2, rows, 2, product_shape(128, R, false, false), (R - k) / 16, false);
            }
            product_commit<1>(&bar);
        }
        made();
        if (mine)
            for (int c = first; c < R; c += 64) {
                float v[16];
                __syncwarp();
                tensor_read(v, at + c);
                if (R > 64) {
                    float t[16];
                    tensor_read(t, at + R + c);
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] += t[k];
                }
                if (row_there) {
                    unsigned char *row = ab + (c >> 6) * L.block + r * 128;
                    ns_add16(row, side, (c >> 3) & 7, r, A.cb, A.cc / kScaleA, v);
                    ns_put16(row, side, (c >> 3) & 7, r, v);
                }
            }
        // up to 512 columns of x at a time
        for (int n0 = 0; n0 < nb; n0 += 8) {
            const int n1 = min(n0 + 8, nb);
            const bool two = R > 64 && n1 - n0 <= 4;       // as many sums as tensor memory has room for
            ready();
            if (tid == 0) {
                for (int b = n0; b < n1; b += 4)
                    for (int k = 0; k < R; k += 64)
                        multiply(acc + (b - n0) * 64 + (two ? (k >> 6) * 256 : 0), desc_rows(abs + (k >> 6) * L.block), 2, desc_columns(xs + b * L.block + k * 128, L.block), 128,
                                 product_shape(128, min(4, n1 - b) * 64, false, true), (R - k) / 16, !two && k > 0);
                product_commit<1>(&bar);
            }
            made();
            if (last) __syncthreads();                   // B may be written over
            if (L.few) {
                // Four of the sixteen warps can read these rows: they pass them on, and all threads do the rest, eight columns of a row
                // each (10 x 4096: 12.6 -> 9.6 us a step).
                float4 *spread = (float4 *)(smem + L.spread);
                if (mine)
                    for (int c = first; c < (n1 - n0) * 64; c += 64) {
                        float v[16];
                        __syncwarp();
                        tensor_read(v, at + c);
                        if (row_there)
#pragma unroll
                            for (int k = 0; k < 4; ++k) spread[(c / 4 + k) * R + r] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                    }
                __syncthreads();
                const int many = (n1 - n0) * 8;
                for (int i = tid; i < many * R; i += kSmallThreads) {
                    // neighbours are rows of a column, or, where they go to a weight with rows of its own, its columns
                    const bool across = last && !tall;
                    const int row = across ? i / many : i % R, ch = across ? i % many : i / R;
                    const float4 a = spread[(2 * ch) * R + row], b = spread[(2 * ch + 1) * R + row];
                    float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    unsigned char *chunk = x + (n0 + (ch >> 3)) * L.block + row * 128 + ((ch ^ row) & 7) * 16;
                    const uint4 hi = *(const uint4 *)chunk;
                    uint4 lo = make_uint4(0, 0, 0, 0);
                    lo = *(const uint4 *)(chunk + side);
                    const uint32_t hs[4] = {hi.x, hi.y, hi.z, hi.w}, ls[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float2 o = __half22float2(*reinterpret_cast<const __half2 *>(&hs[e]));
                        const float2 l = __half22float2(*reinterpret_cast<const __half2 *>(&ls[e]));
                        o.x += l.x;
                        o.y += l.y;
                        v[2 * e] = fmaf(A.ca, o.x, (1.0f / kScaleA) * v[2 * e]);
                        v[2 * e + 1] = fmaf(A.ca, o.y, (1.0f / kScaleA) * v[2 * e + 1]);
                    }
                    if (!last) {
                        uint4 nh, nl;
                        ns_split(v[0], v[1], nh.x, nl.x);
                        ns_split(v[2], v[3], nh.y, nl.y);
                        ns_split(v[4], v[5], nh.z, nl.z);
                        ns_split(v[6], v[7], nh.w, nl.w);
                        *(uint4 *)chunk = nh;
                        *(uint4 *)(chunk + side) = nl;
                    } else {
                        T *dst = (T *)J.dst;
                        const int c0 = (b0 + n0) * 64 + ch * 8;
                        const int64_t to = tall ? (int64_t)c0 * J.cols + row : (int64_t)row * J.cols + c0, step = tall ? J.cols : 1;
                        float w[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] = J.mom && row < J.m && c0 + k < J.n ? ns_in(dst[to + k * step]) : 0.0f;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float o = v[k] * (1.0f / kScaleX);
                            if (row < J.m && c0 + k < J.n) dst[to + k * step] = ns_out<T>(J.mom ? fmaf(J.keep, w[k], -J.step * o) : o);
                        }
                    }
                }
            } else if (mine)
                for (int c = first; c < (n1 - n0) * 64; c += 64) {
                    float v[16];
                    __syncwarp();
                    tensor_read(v, at + c);
                    if (two) {
                        float t[16];
                        tensor_read(t, at + 256 + c);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] += t[k];
                    }
                    const int column = n0 * 64 + c;
                    unsigned char *row = x + (column >> 6) * L.block + r * 128;
                    if (row_there) ns_add16(row, side, (c >> 3) & 7, r, A.ca, 1.0f / kScaleA, v);
                    if (!last) {
                        if (row_there) ns_put16(row, side, (c >> 3) & 7, r, v);
                        continue;
                    }
                    // to the weight: of a tall matrix what the lanes hold of a column, else sixteen elements of two rows at a time
                    T *dst = (T *)J.dst;
                    const int c0 = b0 * 64 + column;
                    float *turned = (float *)(smem + L.scratch) + warp * (32 * 17);
                    if (!tall) {
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 16; ++k) turned[lane * 17 + k] = v[k];
                        __syncwarp();
                    }
                    const int row0 = (warp & 3) * 32;
                    const auto place = [&](int k, int64_t &to) {
                        const int rr = tall ? r : row0 + 2 * k + (lane >> 4), cc = tall ? c0 + k : c0 + (lane & 15);
                        to = tall ? (int64_t)cc * J.cols + rr : (int64_t)rr * J.cols + cc;
                        return rr < J.m && cc < J.n;
                    };
                    float w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        int64_t to;
                        w[k] = place(k, to) && J.mom ? ns_in(dst[to]) : 0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        int64_t to;
                        const float o = (tall ? v[k] : turned[(2 * k + (lane >> 4)) * 17 + (lane & 15)]) * (1.0f / kScaleX);
                        if (place(k, to)) dst[to] = ns_out<T>(J.mom ? fmaf(J.keep, w[k], -J.step * o) : o);
                    }
                }
        }
    }
    if (!fine) atomicExch(status, kStatusNsTimeout);
    tensor_fence_before();
    __syncthreads();
    if (C > 1) cluster_wait_all();
    if (warp == 0) {
        tensor_fence_after();
        tensor_free<1>(acc, 512);
    }
}

static size_t ns_job_bytes(int64_t m, int64_t n)
{
    const int64_t rb = ns_rb((int)m), cbn = ns_cb((int)n);
    return kNormParts * 8 + 256 + (size_t)(2 * rb * cbn + 4 * rb * rb) * (size_t)(kParts * kBlock);
}

// how many matrices of this many bytes a launch takes
static int ns_at_once(int64_t bytes) { return bytes * kMaxJobs <= kMostBytes ? kMaxJobs : bytes <= kMostBytes ? (int)(kMostBytes / bytes) : 1; }

static void ns_take(NsJob &J, unsigned char *&at)
{
    const int64_t rb = ns_rb(J.m), x = rb * ns_cb(J.n) * kParts * kBlock, a = 2 * rb * rb * kParts * kBlock;
    J.parts = (double *)at;
    at += kNormParts * 8 + 256;                  // and a count
    J.x[0] = at;
    J.x[1] = J.x[0] + x;
    J.a = J.x[1] + x;
    J.b = J.a + a;
    at = J.b + a;
}

template <typename T, int MODE>
static int ns_run(NsArgs &A, int steps, cudaStream_t st)
{
    constexpr int CG = NsTile<MODE>::CG;
    NsPlan P = {};
    P.steps = steps;
    P.status = device_status_word();
    if (!P.status) {
        set_error("Newton-Schulz products: no status word on this device");
        return SLAYER_B200_ECUDA;
    }
    P.arrived = (unsigned *)(A.job[0].parts + kNormParts);
    int blocks = 0, m = 0, n = 0;
    for (int j = 0; j < A.jobs; ++j) {
        NsJob &J = A.job[j];
        const int64_t want = ceil_div((int64_t)ns_rb(J.m) * ns_cb(J.n) * 128 * 64, 4096);
        J.norm_parts = (int)(want < kNormParts ? want : kNormParts);
        J.first[0] = blocks;
        J.first[1] = P.tiles[kGram];
        J.first[2] = P.tiles[kUpdate];
        blocks += J.norm_parts;
        const int rt = (ns_rb(J.m) + CG - 1) / CG;
        P.tiles[kGram] += rt * (rt + 1) / 2;
        P.tiles[kUpdate] += rt * ((ns_rb(J.n) + CG - 1) / CG);
        m = J.m > m ? J.m : m;
        n = J.n > n ? J.n : n;
    }
    P.tiles[kPolynomial] = P.tiles[kGram];

    auto kern = ns_steps_kernel<MODE, T>;
    constexpr size_t smem = NsTile<MODE>::kSmem;
    int rc = reserve_dynamic_smem((const void *)kern, smem);
    if (rc) return rc;
    // CTAs that share a tile where there are too few tiles for the SMs, each with two steps of 64 at least.  Five steps with two / four /
    // eight, us: float32 512 x 512 130 / 149 / 173, 2000 x 333 153 / 162 / 173.
    const int least = 4;
    const int index[3] = {ns_cb(n), ns_cb(m), ns_cb(m)};
    int ranks = CG, resident = 0;
    for (int most = MODE == kShared ? 8 : 1;; most = ranks) {
        ranks = CG;
        const int sms = resident ? resident : sm_count();
        for (int k = 0; k < 3; ++k) {
            P.split[k] = 1;
            while (P.split[k] < most && P.tiles[k] * P.split[k] * 2 <= sms && index[k] >= P.split[k] * least) P.split[k] *= 2;
            if (CG == 1) ranks = P.split[k] > ranks ? P.split[k] : ranks;
        }
        const int held = resident_clusters((const void *)kern, ranks, NsTile<MODE>::kThreads, smem) * ranks;
        if (held <= 0) {
            set_error("Newton-Schulz products: the device holds no cluster of %d CTAs", ranks);
            return SLAYER_B200_EUNSUPPORTED;
        }
        const bool settled = resident == held;
        resident = held;
        if (settled || MODE != kShared) break;
    }
    int grid = 0;
    for (int k = 0; k < 3; ++k) {
        const int64_t want = (int64_t)P.tiles[k] * (CG == 2 ? 2 : P.split[k]);
        grid = want < resident ? ((int)want > grid ? (int)want : grid) : resident;
        if (grid == resident) break;
    }
    grid = (int)ceil_div(grid, ranks) * ranks;

    ns_momentum_kernel<T><<<blocks, 256, 0, st>>>(A, P.arrived);
    ns_normalise_kernel<T><<<blocks, 256, 0, st>>>(A);
    rc = check_launch("Newton-Schulz normalisation launch");
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(NsTile<MODE>::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeCooperative;
    attr[1].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kern, A, P);
    return check_launch("Newton-Schulz steps launch");
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

// whether something of this type may lie there
static bool ns_placed(const void *p, int dtype) { return ((uintptr_t)p & (dtype == SLAYER_B200_F32 ? 3 : 1)) == 0; }

// CTAs for each of the small matrices of a launch: up to four column blocks each, more where there are many matrices; 0: a matrix
// does not fit.  Five steps with up to one / two / four / eight blocks, float32, us: 64 x 288 55 / 57 / 59 / 62, 64 x 576 62 / 62 / 65 / 78,
// 100 x 300 94 / 88 / 88 / 85, 20 x 128 x 256 90 / 83 / 69 / 69.
static int ns_small_cluster(const NsArgs &A)
{
    int C = 1;
    for (; C <= 8; C *= 2) {
        bool fits = true, roomy = true;
        for (int j = 0; j < A.jobs && fits; ++j) {
            const int per = ((A.job[j].n + 63) / 64 + C - 1) / C;
            fits = A.job[j].m <= 128 && ns_small(A.job[j].m, per).fits;
            roomy = roomy && per <= 4;
        }
        if (fits && (roomy || C == 8 || A.jobs * C * 2 > sm_count())) return C;
    }
    return 0;
}

template <typename T>
static int ns_run_small(const NsArgs &A, int C, int steps, cudaStream_t st)
{
    int *status = device_status_word();
    if (!status) {
        set_error("Newton-Schulz products: no status word on this device");
        return SLAYER_B200_ECUDA;
    }
    // one CTA per SM, since each takes all of its tensor memory
    size_t smem = 120 * 1024;
    for (int j = 0; j < A.jobs; ++j) {
        const size_t want = 1024 + ns_small(A.job[j].m, ((A.job[j].n + 63) / 64 + C - 1) / C).total;
        smem = want > smem ? want : smem;
    }
    auto kern = ns_small_kernel<T>;
    int rc = reserve_dynamic_smem((const void *)kern, smem);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(A.jobs * C);
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, A, steps, status);
    return check_launch("Newton-Schulz launch for small matrices");
}

template <typename T>
static int ns_tiled(NsArgs &A, int steps, cudaStream_t st)
{
    const int C = ns_small_cluster(A);
    if (C) return ns_run_small<T>(A, C, steps, st);

    // Tiles of two CTAs where there are enough of them; where there are few tiles, CTAs that share them.  Five steps, us, alone / shared /
    // in pairs: float32 512 x 512 170 / 130 / 266, 1024 x 1024 257 / 208 / 373, 1536 x 1536 362 / 368 / 483, 2048 x 2048 586 / 591 / 618,
    // 2304 x 2304 1079 / 1075 / 870
    int64_t tiles = 0;
    for (int j = 0; j < A.jobs; ++j) tiles += (int64_t)((ns_rb(A.job[j].m) + 1) / 2) * ((ns_rb(A.job[j].n) + 1) / 2);
    if (tiles >= sm_count() / 2) return ns_run<T, kPair>(A, steps, st);
    int small = 0;
    for (int j = 0; j < A.jobs; ++j) small += ns_rb(A.job[j].m) * (ns_rb(A.job[j].m) + 1) / 2;
    return small * 4 <= sm_count() ? ns_run<T, kShared>(A, steps, st) : ns_run<T, kAlone>(A, steps, st);
}

static int ns_dispatch(NsArgs &A, int dtype, int steps, cudaStream_t st)
{
    switch (dtype) {
    case SLAYER_B200_F32: return ns_tiled<float>(A, steps, st);
    case SLAYER_B200_BF16: return ns_tiled<__nv_bfloat16>(A, steps, st);
    default: return ns_tiled<__half>(A, steps, st);
    }
}

}  // namespace sb200

using namespace sb200;

extern "C" int64_t slayer_b200_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, int dtype)
{
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    clear_error();
    if (const int rc = ns_shape("orthogonalize", rows, cols)) return rc;
    const int64_t each = (int64_t)ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows), most = ns_at_once(each);
    return each * (batch < most ? batch : most);
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
    SB200_REQUIRE(ns_placed(out, dtype) && ns_placed(in, dtype), "orthogonalize: out and in must be aligned to their elements");
    const size_t bytes = (size_t)rows * cols * (dtype == SLAYER_B200_F32 ? 4 : 2);
    const int most = ns_at_once((int64_t)ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows));
    for (int64_t first = 0; first < batch; first += most) {
        NsArgs A = {};
        A.jobs = (int)(batch - first < most ? batch - first : most);
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
            ns_take(J, at);
        }
        rc = ns_dispatch(A, dtype, steps, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return SLAYER_B200_OK;
}

extern "C" int64_t slayer_b200_muon_step_workspace(const slayer_b200_muon_matrix *list, int64_t count, int dtype)
{
    clear_error();
    int64_t most = 0, now = 0;
    int in = 0;
    for (int64_t i = 0; list && i < count; ++i) {
        const int64_t rows = list[i].rows, cols = list[i].cols;
        if (rows <= 0 || cols <= 0) continue;
        if (const int rc = ns_shape("muon_step", rows, cols)) return rc;
        const int64_t bytes = (int64_t)ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows);
        if (in == kMaxJobs || (in > 0 && now + bytes > kMostBytes)) in = 0, now = 0;       // as slayer_b200_muon_step does
        ++in;
        now += bytes;
        most = now > most ? now : most;
    }
    return most;
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
        SB200_REQUIRE(ns_placed(M.weight, dtype) && ns_placed(M.grad, dtype) && ns_placed(M.momentum, SLAYER_B200_F32),
                      "muon_step: weight, grad and momentum must be aligned to their elements");
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
            const int64_t m = M.rows < M.cols ? M.rows : M.cols, n = M.rows < M.cols ? M.cols : M.rows;
            if (A.jobs > 0 && (at - (unsigned char *)workspace) + (int64_t)ns_job_bytes(m, n) > kMostBytes) break;
            NsJob &J = A.job[A.jobs++];
            J.src = M.grad;
            J.mom = M.momentum;
            J.dst = M.weight;
            J.rows = (int)M.rows;
            J.cols = (int)M.cols;
            J.m = (int)m;
            J.n = (int)n;
            const double r = (double)J.rows / J.cols;
            const double factor = adjust == SLAYER_B200_MUON_SHAPE ? (r > 1.0 ? sqrt(r) : 1.0)
                                : adjust == SLAYER_B200_MUON_RMS   ? 0.2 * sqrt((double)J.n) : 1.0;
            J.keep = (float)(1.0 - (double)lr * (double)weight_decay);
            J.step = (float)((double)lr * factor);
            ns_take(J, at);
        }
        if (A.jobs == 0) break;
        rc = ns_dispatch(A, dtype, steps, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return SLAYER_B200_OK;
}
