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
//   PARTS = 2 (float32, float16 weights): v = hi + lo, two fp16 values, 22 bits and a sign;  v w ~ hi hi + hi lo + lo hi, the
//     left out lo lo being 2^-24 of it.  Three products instead of one, and results as good as fp32 arithmetic's.
//   PARTS = 1 (bfloat16 weights, whose update is rounded to 8 bits in the end): v = hi.
// Sums are fp32 in tensor memory.
//
// X, A and B = b A + c A A live in the workspace as blocks of 128 x 64 elements, padded with zeros, each block laid out as the
// tensor core reads it from shared memory (tensor.cuh), hi before lo: every load is a contiguous copy of 8 to 32 KB, whatever
// the matrix's sizes, and one form of X serves both as rows (X X^T) and as columns (B X).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "tensor.cuh"

namespace sb200 {

constexpr int kMaxJobs = 48;         // matrices per launch
constexpr int kNormParts = 256;      // partial sums of squares per matrix
constexpr int kStatusNsTimeout = 0x5103;
constexpr int kWaitLimit = 1 << 22;
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

// momentum, and the squares' partial sums (double: a sum over up to 2^31 squares, of values of any size)
template <typename T>
__global__ void __launch_bounds__(256) ns_momentum_kernel(const __grid_constant__ NsArgs A)
{
    __shared__ double part[32];
    const NsJob &J = A.job[ns_find<0>(A, blockIdx.x)];
    const int me = blockIdx.x - J.first[0];
    const int64_t count = (int64_t)J.rows * J.cols, step = J.norm_parts * 256ll;
    const T *g = (const T *)J.src;
    double sq = 0.0;
#pragma unroll 4
    for (int64_t i = me * 256ll + threadIdx.x; i < count; i += step) {
        float u = ns_in(g[i]);
        if (J.mom) {
            const float m = fmaf(A.mu, J.mom[i], u);
            J.mom[i] = m;
            u = A.nesterov ? fmaf(A.mu, m, u) : m;
        }
        sq += (double)u * (double)u;
    }
    sq = ns_block_sum(sq, part);
    if (threadIdx.x == 0) J.parts[me] = sq;
}

// two values next to each other as their fp16 parts
template <int PARTS>
__device__ __forceinline__ void ns_split(float v0, float v1, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(v0, v1);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    if (PARTS == 2) {
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(v0 - f.x, v1 - f.y);
        lo = *reinterpret_cast<const uint32_t *>(&l);
    }
}

// where the 16-byte chunk (8 columns from c on) of element (r, c) begins, in blocks of cbs column blocks per row block
template <int PARTS>
__device__ __forceinline__ unsigned char *ns_chunk(unsigned char *x, int cbs, int r, int c)
{
    return x + ((int64_t)(r >> 7) * cbs + (c >> 6)) * (PARTS * kBlock) + (r & 127) * 128 + (((c >> 3) & 7) ^ (r & 7)) * 16;
}

// X0, as blocks: a thread makes a chunk of eight columns
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) ns_normalise_kernel(const __grid_constant__ NsArgs A)
{
    __shared__ double part[32];
    const NsJob &J = A.job[ns_find<0>(A, blockIdx.x)];
    const int me = blockIdx.x - J.first[0];
    const double sq = ns_block_sum((int)threadIdx.x < J.norm_parts ? J.parts[threadIdx.x] : 0.0, part);
    const float inv = (float)((double)kScaleX / (sqrt(sq) + (double)A.eps));
    const T *g = (const T *)J.src;
    const bool tall = J.rows > J.cols;
    const int rows = ns_rb(J.m) * 128, cbs = ns_cb(J.n), chunks = cbs * 8;
    const unsigned total = (unsigned)rows * chunks;           // at most 2^28
    for (unsigned i = me * 256 + threadIdx.x; i < total; i += J.norm_parts * 256) {
        // neighbours in a warp read neighbours in memory: chunks of a row, or (tall) rows of a chunk
        const int r = tall ? (int)(i % (unsigned)rows) : (int)(i / (unsigned)chunks);
        const int c = (int)(tall ? i / (unsigned)rows : i % (unsigned)chunks) * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = 0.0f;
            if (r < J.m && c + k < J.n) {
                const int64_t at = tall ? (int64_t)(c + k) * J.cols + r : (int64_t)r * J.cols + c + k;
                float u = ns_in(g[at]);
                if (J.mom) u = A.nesterov ? fmaf(A.mu, J.mom[at], u) : J.mom[at];
                v[k] = u * inv;
            }
        }
        uint4 hi, lo;
        ns_split<PARTS>(v[0], v[1], hi.x, lo.x);
        ns_split<PARTS>(v[2], v[3], hi.y, lo.y);
        ns_split<PARTS>(v[4], v[5], hi.z, lo.z);
        ns_split<PARTS>(v[6], v[7], hi.w, lo.w);
        unsigned char *at = ns_chunk<PARTS>(J.x[0], cbs, r, c);
        *(uint4 *)at = hi;
        if (PARTS == 2) *(uint4 *)(at + kBlock) = lo;
    }
}

// ------------------------------------------------------------------------------------------------ products
enum NsPhase { kGram, kPolynomial, kUpdate, kLast };

constexpr int kNsThreads = 320;      // a warp that loads, one that issues products, eight that take the results

template <int PARTS, int TN>
struct NsTile {
    static constexpr int kA = PARTS * kBlock, kB = PARTS * kBlock * (TN / 128), kStage = kA + kB;
    static constexpr int kRows = 8 * 32 * 33 * 4;            // one 32 x 32 piece for each of the eight warps
    static constexpr int kStages = (227 * 1024 - 1024 - 512 - kRows) / kStage > 6 ? 6 : (227 * 1024 - 1024 - 512 - kRows) / kStage;
    static constexpr size_t kSmem = 1024 + 512 + kRows + (size_t)kStages * kStage;
};

// Persistent: a CTA takes tiles of 128 x TN of the result.  PHASE
//   kGram        a = x x^T                  kPolynomial  b = cb a + cc a a   (both symmetric: tiles that lie below the diagonal
//   kUpdate      x' = ca x + b x                          are not computed, blocks above it are written twice)
//   kLast        the same, and the result goes to the weight
template <int PHASE, int PARTS, int TN, typename T>
__global__ void __launch_bounds__(kNsThreads, 1) ns_product_kernel(const __grid_constant__ NsArgs A, int from, int tiles, int *status)
{
    using Tile = NsTile<PARTS, TN>;
    constexpr int S = Tile::kStages;
    constexpr bool kSymmetric = PHASE == kGram || PHASE == kPolynomial;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = (uint64_t *)(smem + S * Tile::kStage), *empty = full + S, *done = empty + S, *taken = done + 2;
    uint32_t *base_at = (uint32_t *)(taken + 2);
    float *pieces = (float *)(smem + S * Tile::kStage + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 1) tensor_alloc(base_at, 2 * TN);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(done + i, 1);
            mbar_init(taken + i, 8);
        }
        mbar_init_fence();
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t acc = *base_at;
    bool fine = true;

    // tile -> its job, the row block and the first column block of 128, and how many of those there are
    auto locate = [&](int tile, const NsJob *&J, int &i, int &j, int &nb) {
        const int k = ns_find<kSymmetric ? 1 : 2>(A, tile);
        J = &A.job[k];
        int at = tile - J->first[kSymmetric ? 1 : 2];
        const int rb = ns_rb(J->m), W = TN / 128;
        if (kSymmetric) {
            // row block i has the column tiles from i / W on
            const int ct = (rb + W - 1) / W;
            for (i = 0; at >= ct - i / W; ++i) at -= ct - i / W;
            j = (i / W + at) * W;
            nb = min(W, rb - j);
        } else {
            // tiles that run side by side share columns of x
            i = at % rb;
            j = at / rb * W;
            nb = min(W, ns_rb(J->n) - j);
        }
    };

    if (warp == 0 && lane == 0) {
        int s = 0, phase = 0;
        for (int tile = blockIdx.x; fine && tile < tiles; tile += gridDim.x) {
            const NsJob *J;
            int i, j, nb;
            locate(tile, J, i, j, nb);
            const int cbm = ns_cb(J->m), cbn = ns_cb(J->n);
            const int steps = PHASE == kGram ? cbn : cbm;
            const unsigned char *left = PHASE == kGram ? J->x[from] : PHASE == kPolynomial ? J->a : J->b;
            const unsigned char *right = PHASE == kPolynomial ? J->a : J->x[from];
            const unsigned bytes = PARTS * kBlock * (1 + nb);
            for (int k = 0; k < steps; ++k) {
                if (!mbar_wait_bounded(empty + s, phase ^ 1, kWaitLimit)) { fine = false; break; }
                unsigned char *to = smem + s * Tile::kStage;
                mbar_expect_tx(full + s, bytes);
                bulk_load(to, left + ((int64_t)i * steps + k) * (PARTS * kBlock), PARTS * kBlock, full + s);
                to += Tile::kA;
                if (kSymmetric) {
                    // [part][block]: rows of the operand follow one another
                    for (int b = 0; b < nb; ++b)
                        for (int p = 0; p < PARTS; ++p)
                            bulk_load(to + (p * (TN / 128) + b) * kBlock, right + (((int64_t)(j + b) * steps + k) * PARTS + p) * kBlock, kBlock, full + s);
                } else {
                    // 64 rows of each block of 64 columns: [part][column block]
                    const unsigned char *row = right + ((int64_t)(k >> 1) * cbn + 2 * j) * (PARTS * kBlock) + (k & 1) * (kBlock / 2);
                    for (int b = 0; b < 2 * nb; ++b)
                        for (int p = 0; p < PARTS; ++p)
                            bulk_load(to + (p * (TN / 64) + b) * (kBlock / 2), row + (b * PARTS + p) * kBlock, kBlock / 2, full + s);
                }
                if (++s == S) { s = 0; phase ^= 1; }
            }
        }
        // every stage's last copy has been read before the CTA leaves
        for (int k = 0; k < S; ++k) {
            if (!mbar_wait_bounded(empty + s, phase ^ 1, kWaitLimit)) fine = false;
            if (++s == S) { s = 0; phase ^= 1; }
        }
    } else if (warp == 1 && lane == 0) {
        int s = 0, phase = 0, slot = 0, turn = 0;
        for (int tile = blockIdx.x; fine && tile < tiles; tile += gridDim.x) {
            const NsJob *J;
            int i, j, nb;
            locate(tile, J, i, j, nb);
            const int steps = PHASE == kGram ? ns_cb(J->n) : ns_cb(J->m);
            const uint32_t shape = product_shape(128, nb * 128, !kSymmetric), d = acc + slot * TN;
            if (!mbar_wait_bounded(taken + slot, turn ^ 1, kWaitLimit)) { fine = false; break; }
            tensor_fence_after();
            for (int k = 0; k < steps; ++k) {
                if (!mbar_wait_bounded(full + s, phase, kWaitLimit)) { fine = false; break; }
                tensor_fence_after();
                const unsigned a0 = smem_u32(smem + s * Tile::kStage), b0 = a0 + Tile::kA;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint64_t l[PARTS], r[PARTS];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        l[p] = desc_rows(a0 + p * kBlock + q * 32);
                        r[p] = kSymmetric ? desc_rows(b0 + p * (TN / 128) * kBlock + q * 32)
                                          : desc_columns(b0 + p * (TN / 128) * kBlock + q * 2048, kBlock / 2);
                    }
                    product(d, l[0], r[0], shape, k + q > 0);
                    if (PARTS == 2) {
                        product(d, l[0], r[PARTS - 1], shape, true);
                        product(d, l[PARTS - 1], r[0], shape, true);
                    }
                }
                product_commit(empty + s);
                if (++s == S) { s = 0; phase ^= 1; }
            }
            if (!fine) break;
            product_commit(done + slot);
            if ((slot ^= 1) == 0) turn ^= 1;
        }
        // the results have been taken before the CTA leaves
        for (int k = 0; fine && k < 2; ++k) {
            if (!mbar_wait_bounded(taken + slot, turn ^ 1, kWaitLimit)) fine = false;
            if ((slot ^= 1) == 0) turn ^= 1;
        }
    } else if (warp >= 2) {
        int slot = 0, turn = 0;
        const int w = warp - 2, quarter = warp & 3, half = w >> 2;
        float *piece = pieces + w * 32 * 33;
        for (int tile = blockIdx.x; fine && tile < tiles; tile += gridDim.x) {
            const NsJob *J;
            int i, j, nb;
            locate(tile, J, i, j, nb);
            const int cbm = ns_cb(J->m), cbn = ns_cb(J->n);
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(done + slot, turn, kWaitLimit))) { fine = false; break; }
            tensor_fence_after();
            const int r = i * 128 + quarter * 32 + lane;
            for (int c0 = half * (TN / 2); c0 < (half + 1) * (TN / 2) && c0 < nb * 128; c0 += 32) {
                const int block = j + (c0 >> 7);          // column block of 128
                if (kSymmetric && block < i) continue;
                float v[32];
                tensor_read(v, acc + slot * TN + ((uint32_t)(quarter * 32) << 16) + c0);
                const int c = j * 128 + c0;
                const int cbs = kSymmetric ? cbm : cbn;
                if (PHASE != kGram) {
                    // b = cb a + ..., x' = ca x + ...
                    unsigned char *old = PHASE == kPolynomial ? J->a : J->x[from];
                    const float f = PHASE == kPolynomial ? A.cb : A.ca;
                    const float by = PHASE == kPolynomial ? A.cc / kScaleA : 1.0f / kScaleA;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const unsigned char *at = ns_chunk<PARTS>(old, cbs, r, c + 8 * k);
                        const uint4 hi = *(const uint4 *)at;
                        uint4 lo = make_uint4(0, 0, 0, 0);
                        if (PARTS == 2) lo = *(const uint4 *)(at + kBlock);
                        const uint32_t hs[4] = {hi.x, hi.y, hi.z, hi.w}, ls[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float2 o = __half22float2(*reinterpret_cast<const __half2 *>(&hs[e]));
                            if (PARTS == 2) {
                                const float2 l = __half22float2(*reinterpret_cast<const __half2 *>(&ls[e]));
                                o.x += l.x;
                                o.y += l.y;
                            }
                            v[8 * k + 2 * e] = fmaf(f, o.x, by * v[8 * k + 2 * e]);
                            v[8 * k + 2 * e + 1] = fmaf(f, o.y, by * v[8 * k + 2 * e + 1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] *= kScaleA / (kScaleX * kScaleX);
                }
                if (PHASE == kLast) {
                    // to the weight, 32 elements next to each other at a time: of a tall matrix, what the lanes hold of a column
                    T *dst = (T *)J->dst;
                    const auto put = [&](int row, int col, int64_t at, float o) {
                        o *= 1.0f / kScaleX;
                        if (row < J->m && col < J->n) dst[at] = ns_out<T>(J->mom ? fmaf(J->keep, ns_in(dst[at]), -J->step * o) : o);
                    };
                    if (J->rows > J->cols) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) put(r, c + k, (int64_t)(c + k) * J->cols + r, v[k]);
                    } else {
                        const int r0 = i * 128 + quarter * 32;
#pragma unroll
                        for (int k = 0; k < 32; ++k) piece[lane * 33 + k] = v[k];
                        __syncwarp();
#pragma unroll 8
                        for (int k = 0; k < 32; ++k) put(r0 + k, c + lane, (int64_t)(r0 + k) * J->cols + c + lane, piece[k * 33 + lane]);
                    }
                    __syncwarp();
                    continue;
                }
                unsigned char *to = PHASE == kGram ? J->a : PHASE == kPolynomial ? J->b : J->x[from ^ 1];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint4 hi, lo;
                    ns_split<PARTS>(v[8 * k], v[8 * k + 1], hi.x, lo.x);
                    ns_split<PARTS>(v[8 * k + 2], v[8 * k + 3], hi.y, lo.y);
                    ns_split<PARTS>(v[8 * k + 4], v[8 * k + 5], hi.z, lo.z);
                    ns_split<PARTS>(v[8 * k + 6], v[8 * k + 7], hi.w, lo.w);
                    unsigned char *at = ns_chunk<PARTS>(to, cbs, r, c + 8 * k);
                    *(uint4 *)at = hi;
                    if (PARTS == 2) *(uint4 *)(at + kBlock) = lo;
                    if (kSymmetric && block > i) {
                        // (c, r) too: 32 lanes write 64 bytes of a row
                        const uint32_t hs[4] = {hi.x, hi.y, hi.z, hi.w}, ls[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            unsigned char *mirror = ns_chunk<PARTS>(to, cbs, c + 8 * k + e, r) + (r & 7) * 2;
                            *(uint16_t *)mirror = (uint16_t)(hs[e >> 1] >> (e & 1) * 16);
                            if (PARTS == 2) *(uint16_t *)(mirror + kBlock) = (uint16_t)(ls[e >> 1] >> (e & 1) * 16);
                        }
                    }
                }
            }
            tensor_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(taken + slot);
            if ((slot ^= 1) == 0) turn ^= 1;
        }
    }
    if (!fine) atomicExch(status, kStatusNsTimeout);
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    if (warp == 1) {
        tensor_fence_after();
        tensor_free(acc, 2 * TN);
    }
}

static size_t ns_job_bytes(int64_t m, int64_t n, int dtype)
{
    const int64_t parts = dtype == SLAYER_B200_BF16 ? 1 : 2, rb = ns_rb((int)m), cbn = ns_cb((int)n);
    return kNormParts * 8 + (size_t)(2 * rb * cbn + 4 * rb * rb) * (size_t)(parts * kBlock);
}

static void ns_take(NsJob &J, int parts, unsigned char *&at)
{
    const int64_t rb = ns_rb(J.m), x = rb * ns_cb(J.n) * parts * kBlock, a = 2 * rb * rb * parts * kBlock;
    J.parts = (double *)at;
    at += kNormParts * 8;
    J.x[0] = at;
    J.x[1] = J.x[0] + x;
    J.a = J.x[1] + x;
    J.b = J.a + a;
    at = J.b + a;
}

template <int PHASE, int PARTS, int TN, typename T>
static int ns_product(const NsArgs &A, int from, int tiles, int *status, cudaStream_t st)
{
    auto kern = ns_product_kernel<PHASE, PARTS, TN, T>;
    constexpr size_t smem = NsTile<PARTS, TN>::kSmem;
    int rc = reserve_dynamic_smem((const void *)kern, smem);
    if (rc) return rc;
    kern<<<tiles < sm_count() ? tiles : sm_count(), kNsThreads, smem, st>>>(A, from, tiles, status);
    return check_launch("Newton-Schulz product launch");
}

template <typename T, int PARTS, int TN>
static int ns_run(NsArgs &A, int steps, cudaStream_t st)
{
    int *status = device_status_word();
    if (!status) {
        set_error("Newton-Schulz products: no status word on this device");
        return SLAYER_B200_ECUDA;
    }
    int blocks = 0, small = 0, large = 0;
    for (int j = 0; j < A.jobs; ++j) {
        NsJob &J = A.job[j];
        const int64_t want = ceil_div((int64_t)ns_rb(J.m) * ns_cb(J.n) * 128 * 64, 4096);
        J.norm_parts = (int)(want < kNormParts ? want : kNormParts);
        J.first[0] = blocks;
        J.first[1] = small;
        J.first[2] = large;
        blocks += J.norm_parts;
        const int rb = ns_rb(J.m), W = TN / 128, ct = (rb + W - 1) / W;
        for (int i = 0; i < rb; ++i) small += ct - i / W;
        large += rb * ((ns_rb(J.n) + W - 1) / W);
    }
    ns_momentum_kernel<T><<<blocks, 256, 0, st>>>(A);
    int rc = check_launch("momentum launch");
    if (rc) return rc;
    int from = 0;
    ns_normalise_kernel<T, PARTS><<<blocks, 256, 0, st>>>(A);
    rc = check_launch("Newton-Schulz normalisation launch");
    for (int s = 0; s < steps && !rc; ++s, from ^= 1) {
        rc = ns_product<kGram, PARTS, TN, float>(A, from, small, status, st);
        if (!rc) rc = ns_product<kPolynomial, PARTS, TN, float>(A, from, small, status, st);
        if (!rc) rc = s + 1 < steps ? ns_product<kUpdate, PARTS, TN, float>(A, from, large, status, st)
                                    : ns_product<kLast, PARTS, TN, T>(A, from, large, status, st);
    }
    return rc;
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

template <typename T, int PARTS>
static int ns_tiled(NsArgs &A, int steps, cudaStream_t st)
{
    // wide tiles where there are enough of them
    int64_t tiles = 0;
    for (int j = 0; j < A.jobs; ++j) tiles += (int64_t)ns_rb(A.job[j].m) * ns_rb(A.job[j].m) / 4;
    return tiles >= sm_count() ? ns_run<T, PARTS, 256>(A, steps, st) : ns_run<T, PARTS, 128>(A, steps, st);
}

static int ns_dispatch(NsArgs &A, int dtype, int steps, cudaStream_t st)
{
    switch (dtype) {
    case SLAYER_B200_F32: return ns_tiled<float, 2>(A, steps, st);
    case SLAYER_B200_BF16: return ns_tiled<__nv_bfloat16, 1>(A, steps, st);
    default: return ns_tiled<__half, 2>(A, steps, st);
    }
}

}  // namespace sb200

using namespace sb200;

extern "C" int64_t slayer_b200_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, int dtype)
{
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    return (int64_t)ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows, dtype) * (batch < kMaxJobs ? batch : kMaxJobs);
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
            ns_take(J, dtype == SLAYER_B200_BF16 ? 1 : 2, at);
        }
        rc = ns_dispatch(A, dtype, steps, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return SLAYER_B200_OK;
}

extern "C" int64_t slayer_b200_muon_step_workspace(const slayer_b200_muon_matrix *list, int64_t count, int dtype)
{
    size_t most = 0, now = 0;
    int in = 0;
    for (int64_t i = 0; list && i < count; ++i) {
        const int64_t rows = list[i].rows, cols = list[i].cols;
        if (rows <= 0 || cols <= 0) continue;
        if (in++ == kMaxJobs) {
            in = 1;
            now = 0;
        }
        now += ns_job_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows, dtype);
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
            ns_take(J, dtype == SLAYER_B200_BF16 ? 1 : 2, at);
        }
        if (A.jobs == 0) break;
        rc = ns_dispatch(A, dtype, steps, (cudaStream_t)stream);
        if (rc) return rc;
    }
    return SLAYER_B200_OK;
}
