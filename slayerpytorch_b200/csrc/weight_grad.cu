// Weight gradient of a dense layer from an input kept in 8 bits (checkpoint.cu):
//   dW[o, i] = sum over samples n and steps t of g[n, o, t] x[n, i, t],  x = q 2^e,
// as products of bfloat16 tiles on the tensor cores.  q 2^e is a bfloat16 as it is; g, a float32, is the sum of three: its upper 8 bits, the
// next 8 and the last 8, cut off and not rounded, so that the three parts are g exactly (but for what is below 2^-133, bfloat16's smallest number: a g
// under 2^-110 has bits there).  What is not finite leaves parts that are NaN.  Three products, summed in float32, have the
// precision of float32 products.  Both operands have time as their summation index and next to each other in memory, as the tensor cores
// like it, but neither is in a form that they read: 16 warps fetch tiles (16-byte copies to shared memory that nobody waits for, two blocks
// ahead), take them apart in registers and write them to shared memory again as 128-byte rows; one thread issues the products.
//
// The tensor core cuts sums off where it adds: sums of kSteps blocks of 64 steps are made there, and added up in registers, rounded.
//
// x is the operand with the tile's rows (i), g the one with its columns (o): large layers take tiles of 256 x 256 by pairs of CTAs, each of which loads and
// takes apart one half of either; layers of up to 128 outputs tiles of 128 x 16 to 128 x 128 by one CTA.  The tiles' blocks of 64 steps are dealt out
// to all SMs in equal shares (tile after tile: a share has the end of one tile, some whole ones and the start of another), and the shares'
// sums are added up by a second launch, in order.  Its CTAs start as the first launch's leave, and wait there for the last of them (2 us less than one
// launch after the other, at every size).
#include <algorithm>

#include "tensor.cuh"

namespace sb200 {

constexpr int kWgWaitLimit = 1 << 22;
constexpr int kStatusWeightTimeout = 0x5104;
constexpr int kWgWorkers = 512, kWgThreads = kWgWorkers + 128;
constexpr int kSteps = 2;        // blocks of 64 steps in a sum of the tensor core (4: 1.5 % faster, results twice as far off)

template <int CG, int NT, bool VEC>
struct WgTile {
    static constexpr int NB = NT / CG;                      // columns (of g) that a CTA loads
    static constexpr int kA = 128 * 128, kB = NB * 128;     // bytes of a block of 64 steps: x, and one part of g
    static constexpr int kStage = kA + 3 * kB;
    static constexpr int kCols = NT >= 64 ? NT / 4 : 16;    // of a warp's sums
    static constexpr int kItems = NB >= 32 ? NB / 32 : 1;   // float4 of g a thread has of a block
    static constexpr uint32_t kMem = 2 * NT;
    // as fetched: a thread's 16 bytes of x, its float4s of g, and those after them
    static constexpr int kRaw = (1 + kItems) * kWgWorkers * 16 + (VEC ? 0 : kItems * kWgWorkers / 4 * 16);
    static constexpr int kStages = (225 * 1024 - 2 * kRaw) / kStage < 4 ? (225 * 1024 - 2 * kRaw) / kStage : 4;
    static constexpr size_t kShared = kStages * kStage + 2 * kRaw + 1024;
    static_assert(kStages >= 2 && kShared <= 226 * 1024, "shared memory");
};

struct WgArgs {
    const float *g;
    const int8_t *q;
    const uint8_t *scale;
    float *part;
    int *status;
    int64_t N, O, I, T, G, g_size;
    int units, blocks, U;        // 16 steps of a sample; 4 of those; units of a sample
    int inner_samples;           // samples with at least eight elements of g behind them
    int64_t tiles_o, work;       // tiles next to each other share their rows; tiles x blocks
    int shares;
};

// A 16-step unit that a thread has, and the ones four further on.
struct WgUnit {
    int unit, n, t16;
    __device__ __forceinline__ void start(int u, int U)
    {
        unit = u;
        n = u / U;
        t16 = u - n * U;
    }
    // true: of another sample
    __device__ __forceinline__ bool next(int U)
    {
        unit += 4;
        t16 += 4;
        if (t16 < U) return false;
        do {
            t16 -= U;
            ++n;
        } while (t16 >= U);
        return true;
    }
};

// the upper 16 bits of two floats
__device__ __forceinline__ uint32_t upper(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ float cut(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }

// 16 bytes on their way to shared memory, zeros behind the first `bytes`
__device__ __forceinline__ void wg_copy(void *to, const void *from, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void wg_copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wg_copies_wait() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void wg_copies_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// the four of a's and b's eight that begin `skew` behind a's first, zeros behind the first `left`
__device__ __forceinline__ float4 wg_shift(float4 a, float4 b, int skew, int left)
{
    const bool two = skew & 2, one = skew & 1;
    const float v0 = two ? a.z : a.x, v1 = two ? a.w : a.y, v2 = two ? b.x : a.z, v3 = two ? b.y : a.w, v4 = two ? b.z : b.x;
    float4 v = make_float4(one ? v1 : v0, one ? v2 : v1, one ? v3 : v2, one ? v4 : v3);
    if (left < 4) {
        v.x = left > 0 ? v.x : 0.0f;
        v.y = left > 1 ? v.y : 0.0f;
        v.z = left > 2 ? v.z : 0.0f;
        v.w = 0.0f;
    }
    return v;
}

// two floats at once: a b + c
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// what is left of two floats without their upper 16 bits
__device__ __forceinline__ float2 rest2(float2 v) { return fma2(make_float2(cut(v.x), cut(v.y)), make_float2(-1.0f, -1.0f), v); }

// 16 whole numbers times a power of two, as bfloat16
__device__ __forceinline__ void wg_expand(uint4 raw, unsigned byte, uint4 &lo, uint4 &hi)
{
    constexpr float kBias = 8388608.0f + 128.0f;
    const uint32_t w[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};     // q + 128
    uint32_t none = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) none |= (w[k] - 0x01010101u) & ~w[k];      // a byte of 0: q is -128, what was not finite
    // 2^23 + q + 128 as the float that ends in that byte, times the scale, minus (2^23 + 128) times it: exact, unless that is too large
    const float s = __uint_as_float(byte << 23);
    uint32_t out[8];
    if (!(none & 0x80808080u) && byte < 220) {
        const float2 s2 = make_float2(s, s), c2 = make_float2(-kBias * s, -kBias * s);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 v = make_float2(__uint_as_float(__byte_perm(w[k / 2], 0x4b000000u, 0x7540 | (k & 1) * 2)),
                                         __uint_as_float(__byte_perm(w[k / 2], 0x4b000000u, 0x7541 | (k & 1) * 2)));
            const float2 f = fma2(v, s2, c2);
            out[k] = upper(f.x, f.y);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int q0 = (int)((w[k / 2] >> ((k & 1) * 16)) & 0xff) - 128, q1 = (int)((w[k / 2] >> ((k & 1) * 16 + 8)) & 0xff) - 128;
            out[k] = upper(q0 == -128 ? __uint_as_float(0x7fc00000u) : (float)q0 * s, q1 == -128 ? __uint_as_float(0x7fc00000u) : (float)q1 * s);
        }
    }
    lo = make_uint4(out[0], out[1], out[2], out[3]);
    hi = make_uint4(out[4], out[5], out[6], out[7]);
}

template <int CG, int NT, bool VEC>
__global__ void __launch_bounds__(kWgThreads, 1) weight_grad_kernel(const __grid_constant__ WgArgs A)
{
    using Tile = WgTile<CG, NT, VEC>;
    constexpr int S = Tile::kStages, kItems = Tile::kItems;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[S], empty[S], made[2], taken[2], last;
    __shared__ uint32_t base_at;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CG == 2 ? (int)cluster_rank() : 0;
    const int share = blockIdx.x / CG;
    const int64_t from = A.work * share / A.shares, to = A.work * (share + 1) / A.shares;
    uint32_t acc = 0;
    bool fine = true;
    // barriers and tensor memory are there: what the workers wait for with their first blocks on the way
    const auto ready = [&] {
        tensor_fence_before();
        asm volatile("barrier.cta.sync 1, %0;" ::"n"(kWgThreads) : "memory");
        if (CG == 2) cluster_wait_all();
        tensor_fence_after();
        acc = base_at;
    };

    // registers: 512 * 112 + 128 * 32 = 640 * 96
    if (warp < 16) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        // x: a row and one of the four units; g: rows of 8 (in an order that keeps the stores of a half warp on different banks), one unit
        const int arow = warp * 8 + (lane >> 2), au = lane & 3, quarter = lane & 3, bu = warp & 3;
        const int brow = (warp >> 2) * (Tile::NB >= 32 ? Tile::NB / 4 : 8) + 2 * ((lane >> 2) & 3) + (lane >> 4);
        const bool has_b = Tile::NB >= 32 || (warp >> 2) * 8 < Tile::NB;
        const bool sums_here = (warp >> 2) * Tile::kCols < NT;
        // what a thread has fetched lies where nobody else (VEC), or nobody else of another warp, reads it
        unsigned char *const raw = smem + S * Tile::kStage + tid * 16;
        // what comes after them, where the next thread does not have it: for one of the four threads of a row's unit
        const unsigned beyond = (1 + kItems) * 8192 - tid * 16 + (tid >> 2) * 16;

        // The block after next, on its way.  Rows behind the last are the last once more: their results are nobody's.  Steps behind the last are zeros.
        int64_t ahead = from;
        int tile_left = 0;              // blocks
        const int8_t *aq = A.q;         // this thread's unit
        const uint8_t *as = A.scale;
        const float *bg = A.g;
        int b_far[kItems];              // its rows of g from the first one on
        WgUnit ua = {}, ub = {};
        unsigned scale_0 = 127, scale_1 = 127;
        int64_t i = 0, o = 0;
        const auto find_a = [&] {
            aq = A.q + ((int64_t)ua.n * A.I + i) * (A.G * 32) + ua.t16 * 16;
            as = A.scale + ((ua.t16 >> 1) * A.N + ua.n) * A.I + i;
        };
        const auto find_b = [&] { bg = A.g + ((int64_t)ub.n * A.O + o) * A.T + ub.t16 * 16 + quarter * 4; };
        const int64_t a_groups = 2 * A.N * A.I;
        const auto fetch = [&](int slot, unsigned &scale) {
            if (ahead < to) {
                if (tile_left == 0) {
                    const int64_t tile = ahead / A.blocks, ti = tile / A.tiles_o;
                    const int k = (int)(ahead - tile * A.blocks);
                    tile_left = A.blocks - k;
                    i = min((ti * CG + rank) * 128 + arow, A.I - 1);
                    o = min((tile - ti * A.tiles_o) * NT + rank * Tile::NB + brow, A.O - 1);
                    const int last = (int)min((A.O - 1 - o) / 8, (int64_t)kItems - 1);
#pragma unroll
                    for (int j = 0; j < kItems; ++j) b_far[j] = min(j, last) * 8 * (int)A.T;
                    ua.start(k * 4 + au, A.U);
                    ub.start(k * 4 + bu, A.U);
                    find_a();
                    find_b();
                }
                unsigned char *const into = raw + slot * Tile::kRaw;
                const bool a = ua.unit < A.units;
                wg_copy(into, a ? aq : A.q, a ? 16 : 0);
                if (a) scale = __ldg(as);
                if (has_b) {
                    const int t = ub.t16 * 16 + quarter * 4;
                    const bool b = ub.unit < A.units && t < (int)A.T;
                    if (VEC) {
#pragma unroll
                        for (int j = 0; j < kItems; ++j) wg_copy(into + (1 + j) * 8192, b ? bg + b_far[j] : A.g, b ? 16 : 0);
                    } else {
                        // The 16 bytes that the four steps begin in, and, where the thread beside has no more steps of the row or a quarter is the
                        // unit's last, the 16 after them.  The tensor may end inside.
                        const float *const p = b ? bg - ((int)(bg - A.g) & 3) : A.g;
                        const bool more = b && (quarter == 3 || t + 4 >= (int)A.T);
                        if (ub.n < A.inner_samples) {
#pragma unroll
                            for (int j = 0; j < kItems; ++j) {
                                const float *v = p + (b ? b_far[j] : 0);
                                wg_copy(into + (1 + j) * 8192, v, b ? 16 : 0);
                                if (more) wg_copy(into + beyond + j * 2048, v + 4, 16);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < kItems; ++j) {
                                const float *v = p + (b ? b_far[j] : 0);
                                const int there = (int)min(A.g_size - (v - A.g), (int64_t)8);
                                wg_copy(into + (1 + j) * 8192, v, b ? min(there * 4, 16) : 0);
                                if (more) wg_copy(into + beyond + j * 2048, there > 4 ? v + 4 : v, max(there * 4 - 16, 0));
                            }
                        }
                    }
                }
                ++ahead;
                --tile_left;
                // the next unit: mostly the same sample's, two groups of steps on
                aq += 64;
                as += a_groups;
                bg += 64;
                if (ua.next(A.U)) find_a();
                if (ub.next(A.U)) find_b();
            }
            wg_copies_commit();
        };
        int s = 0, turn = 0, slot = 0, again = 0, from_slot = 0;
        fetch(0, scale_0);
        fetch(1, scale_1);
        ready();
        const uint32_t at = acc + ((uint32_t)((warp & 3) * 32) << 16) + (warp >> 2) * Tile::kCols;
        WgUnit uc;        // of g in the block that is worked on: what lies behind T is not g's
        for (int64_t w = from; fine && w < to;) {
            const int64_t tile = w / A.blocks;
            const int k0 = (int)(w - tile * A.blocks), k1 = (int)min((int64_t)A.blocks, k0 + (to - w));
            float sum[Tile::kCols];
#pragma unroll
            for (int k = 0; k < Tile::kCols; ++k) sum[k] = 0.0f;
            const auto take = [&] {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(made + slot, again, kWgWaitLimit))) {
                    fine = false;
                    return;
                }
                tensor_fence_after();
                if (sums_here) {
                    constexpr int kPiece = 16;
#pragma unroll
                    for (int c = 0; c < Tile::kCols; c += kPiece) {
                        float v[kPiece];
                        tensor_read(v, at + slot * NT + c);
#pragma unroll
                        for (int k = 0; k < kPiece; k += 2) {
                            const float2 two = add2(make_float2(sum[c + k], sum[c + k + 1]), make_float2(v[k], v[k + 1]));
                            sum[c + k] = two.x;
                            sum[c + k + 1] = two.y;
                        }
                    }
                }
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) mbar_arrive_at(taken + slot, 0);
                    else mbar_arrive(taken + slot);
                }
                if ((slot ^= 1) == 0) again ^= 1;
            };
            if (!VEC) uc.start(k0 * 4 + bu, A.U);
            const unsigned o = (unsigned)min((tile % A.tiles_o) * NT + rank * Tile::NB + brow, A.O - 1);
            int groups = 0;        // sums that have been taken
            for (int k = k0; k < k1; ++k) {
                wg_copies_wait();
                if (!VEC) __syncwarp();
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(empty + s, turn ^ 1, kWgWaitLimit))) { fine = false; break; }
                const unsigned char *const in = raw + from_slot * Tile::kRaw;
                unsigned char *const a = smem + s * Tile::kStage + arow * 128;
                unsigned char *const b = smem + s * Tile::kStage + Tile::kA + brow * 128 + (((2 * bu + (quarter >> 1)) ^ (brow & 7)) * 16) + (quarter & 1) * 8;
                {
                    uint4 lo, hi;
                    wg_expand(*(const uint4 *)in, scale_0, lo, hi);
                    *(uint4 *)(a + (((2 * au) ^ arow) & 7) * 16) = lo;
                    *(uint4 *)(a + (((2 * au + 1) ^ arow) & 7) * 16) = hi;
                }
                if (has_b) {
                    int skew = 0, left = 4;
                    bool more = false;
                    if (!VEC) {
                        const int t = uc.t16 * 16 + quarter * 4;
                        skew = (int)(((unsigned)uc.n * (unsigned)A.O + o) * (unsigned)A.T & 3u);        // (8 rows on it is the same)
                        left = uc.unit < A.units ? (int)min(A.T - t, (int64_t)4) : 0;
                        more = quarter == 3 || t + 4 >= A.T;
                    }
#pragma unroll
                    for (int j = 0; j < kItems; ++j) {
                        float4 v = *(const float4 *)(in + (1 + j) * 8192);
                        if (!VEC) v = wg_shift(v, *(const float4 *)(in + (more ? beyond + j * 2048 : (1 + j) * 8192 + 16)), skew, left);
                        const float2 u = rest2(make_float2(v.x, v.y)), w = rest2(make_float2(v.z, v.w)), x = rest2(u), y = rest2(w);
                        *(uint2 *)(b + j * 1024) = make_uint2(upper(v.x, v.y), upper(v.z, v.w));
                        *(uint2 *)(b + Tile::kB + j * 1024) = make_uint2(upper(u.x, u.y), upper(w.x, w.y));
                        *(uint2 *)(b + 2 * Tile::kB + j * 1024) = make_uint2(upper(x.x, x.y), upper(y.x, y.y));
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) mbar_arrive_at(full + s, 0);
                    else mbar_arrive(full + s);
                }
                if (++s == S) { s = 0; turn ^= 1; }
                scale_0 = scale_1;
                fetch(from_slot, scale_1);
                from_slot ^= 1;
                if (!VEC) uc.next(A.U);
                // the sum before the one whose last block this is: its products are done, or nearly so
                const int done = k - k0 + 1;
                if (done % kSteps == 0 && done / kSteps >= 2) {
                    take();
                    ++groups;
                    if (!fine) break;
                }
            }
            for (const int all = (k1 - k0 + kSteps - 1) / kSteps; fine && groups < all; ++groups) take();
            if (fine && sums_here) {
                // the part of this share and tile: [column][row]
                float *out = A.part + (share + tile) * (int64_t)(128 * CG * NT) + (int64_t)((warp >> 2) * Tile::kCols) * (128 * CG) + rank * 128 + (warp & 3) * 32 + lane;
#pragma unroll
                for (int k = 0; k < Tile::kCols; ++k) out[k * (128 * CG)] = sum[k];
            }
            w += k1 - k0;
        }
        wg_copies_wait_all();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        if (warp == 16) tensor_alloc<CG>(&base_at, Tile::kMem);
        if (tid == kWgWorkers) {
            for (int s = 0; s < S; ++s) {
                mbar_init(full + s, 16 * CG);
                mbar_init(empty + s, 1);
            }
            for (int b = 0; b < 2; ++b) {
                mbar_init(made + b, 1);
                mbar_init(taken + b, 16 * CG);
            }
            mbar_init(&last, 1);
            mbar_init_fence();
        }
        __syncwarp();
        ready();
    }
    if (warp == 16 && lane == 0 && rank == 0) {
        constexpr uint32_t kShape = product_shape_bf16(128 * CG, NT);
        int s = 0, turn = 0, slot = 0, again = 0;
        for (int64_t w = from; fine && w < to;) {
            const int n = (int)min(A.blocks - w % A.blocks, to - w);
            for (int k = 0; k < n; ++k) {
                const bool first = k % kSteps == 0;
                if (first && !mbar_wait_bounded(taken + slot, again ^ 1, kWgWaitLimit)) { fine = false; break; }
                if (!mbar_wait_bounded(full + s, turn, kWgWaitLimit)) { fine = false; break; }
                tensor_fence_after();
                const unsigned a0 = smem_u32(smem + s * Tile::kStage), b0 = a0 + Tile::kA;
                const uint64_t a = desc_rows(a0);
                // the small parts first: what they lose to the sum's size is less while it is small
#pragma unroll
                for (int part = 2; part >= 0; --part) {
                    const uint64_t b = desc_rows(b0 + part * Tile::kB);
#pragma unroll
                    for (int j = 0; j < 4; ++j) product<CG>(acc + slot * NT, a + 2 * j, b + 2 * j, kShape, !(first && part == 2 && j == 0));
                }
                product_commit<CG>(empty + s);
                if (++s == S) { s = 0; turn ^= 1; }
                if ((k + 1) % kSteps == 0 || k + 1 == n) {
                    product_commit<CG>(made + slot);
                    if ((slot ^= 1) == 0) again ^= 1;
                }
            }
            w += n;
        }
        product_commit<CG>(&last);
    }
    // the CTAs that add the parts up may take the place of this one
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // all products have read their operands, and told so, before a CTA leaves
    if (warp == 16 && lane == 0 && !mbar_wait_bounded(&last, 0, kWgWaitLimit)) fine = false;
    __syncwarp();
    if (!fine) atomicExch(A.status, kStatusWeightTimeout);
    tensor_fence_before();
    __syncthreads();
    if (CG == 2) cluster_wait_all();
    if (warp == 16) {
        tensor_fence_after();
        tensor_free<CG>(acc, Tile::kMem);
    }
}

// The shares' parts of each output, in order: SPLIT warps have 128 rows of a column, four of them a thread, and every SPLIT-th part.
template <int CG, int NT, int SPLIT>
__global__ void __launch_bounds__(256) weight_sum_kernel(float *out, const WgArgs A)
{
    constexpr int R = 128 * CG;
    __shared__ int range[2];
    __shared__ double sums[SPLIT > 1 ? 8 : 1][4][32];
    const int64_t tile = blockIdx.x, ti = tile / A.tiles_o, to = tile - ti * A.tiles_o;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y * 128 + lane * 4;
    const int col = blockIdx.z * (8 / SPLIT) + warp / SPLIT, turn = warp % SPLIT;
    // share p begins at work * p / shares: the one that has a block is the last to begin before or at it
    if (threadIdx.x < 2) range[threadIdx.x] = (int)((((tile + threadIdx.x) * A.blocks + 1 - threadIdx.x) * A.shares - 1) / A.work);
    __syncthreads();
    const int first = range[0], last = range[1];
    asm volatile("griddepcontrol.wait;" ::: "memory");       // all parts are there
    const int64_t i = ti * R + row, o = to * NT + col;
    const bool there = i < A.I && o < A.O;
    double sum[4] = {};
    const float *p = A.part + (first + turn + tile) * (int64_t)(R * NT) + (int64_t)col * R + row;
#pragma unroll 8
    for (int s = first + turn; s <= last && there; s += SPLIT, p += SPLIT * (int64_t)(R * NT)) {
        const float4 v = *reinterpret_cast<const float4 *>(p);        // (__ldg might be moved before the wait)
        sum[0] += (double)v.x, sum[1] += (double)v.y, sum[2] += (double)v.z, sum[3] += (double)v.w;
    }
    if (SPLIT > 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[warp][k][lane] = sum[k];
        __syncthreads();
#pragma unroll
        for (int w = 1; w < SPLIT; ++w)
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] += sums[(warp - turn + w) & 7][k][lane];
    }
    if (!there || turn > 0) return;
    float *to_row = out + o * A.I + i;
    if (A.I % 4 == 0 && ((uintptr_t)out & 15) == 0) {
        *reinterpret_cast<float4 *>(to_row) = make_float4((float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < A.I) to_row[k] = (float)sum[k];
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct WgPlan {
    int cg, nt;
    int64_t tiles, tiles_o, blocks, shares;
    int64_t bytes;
};

static WgPlan wg_plan(int64_t N, int64_t O, int64_t I, int64_t T)
{
    WgPlan p;
    // a pair's tile of 256 outputs where there are more than 128; else the smallest tile that has them all
    p.cg = O > 128 ? 2 : 1;
    p.nt = O > 128 ? 256 : O > 64 ? 128 : O > 32 ? 64 : O > 16 ? 32 : 16;
    p.tiles_o = ceil_div(O, p.nt);
    p.tiles = p.tiles_o * ceil_div(I, 128 * p.cg);
    p.blocks = ceil_div(N * ceil_div(T, 16), 4);
    // a share has four blocks at least: less is not worth its part of the sum
    const int64_t most = sm_count() / p.cg, work = p.tiles * p.blocks;
    p.shares = std::max<int64_t>(1, std::min(most, ceil_div(work, 4)));
    p.bytes = (p.tiles + p.shares) * (int64_t)(128 * p.cg * p.nt) * 4;
    return p;
}

static int wg_check(const char *op, int64_t N, int64_t O, int64_t I, int64_t T)
{
    SB200_REQUIRE(N >= 0 && O >= 0 && I >= 0 && T >= 0, "%s: negative size", op);
    const int64_t most = (int64_t)1 << 31;
    SB200_REQUIRE(N < most && O <= (int64_t)1 << 22 && I < most && T <= (int64_t)1 << 26, "%s: sizes are too large", op);
    SB200_REQUIRE(N * ceil_div(T, 16) < most - 64 && (O >> 7) * (I >> 7) < (int64_t)1 << 22, "%s: sizes are too large", op);
    return SLAYER_B200_OK;
}

template <int CG, int NT, bool VEC>
static int wg_launch(const WgArgs &A, float *out, int64_t tiles, cudaStream_t st)
{
    using Tile = WgTile<CG, NT, VEC>;
    auto kern = weight_grad_kernel<CG, NT, VEC>;
    const int rc = reserve_dynamic_smem((const void *)kern, Tile::kShared);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(A.shares * CG));
    cfg.blockDim = dim3(kWgThreads);
    cfg.dynamicSmemBytes = Tile::kShared;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, A);
    const int bad = check_launch("weight_grad8 kernel launch");
    if (bad) return bad;
    // (a tile with many parts: 37 of them one after the other 7.5 us, in fours 4.7)
    const bool many = A.shares / tiles >= 16;
    cudaLaunchConfig_t then = {};
    then.gridDim = dim3((unsigned)tiles, CG, many ? NT / 2 : NT / 8);
    then.blockDim = dim3(256);
    then.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    then.attrs = attr;
    then.numAttrs = 1;
    cudaLaunchKernelEx(&then, many ? weight_sum_kernel<CG, NT, 4> : weight_sum_kernel<CG, NT, 1>, out, A);
    return check_launch("weight_grad8 sum launch");
}

template <int CG, int NT>
static int wg_align(const WgArgs &A, float *out, int64_t tiles, cudaStream_t st)
{
    return A.T % 4 == 0 ? wg_launch<CG, NT, true>(A, out, tiles, st) : wg_launch<CG, NT, false>(A, out, tiles, st);
}

}  // namespace sb200

extern "C" int64_t slayer_b200_weight_grad8_workspace(int64_t N, int64_t O, int64_t I, int64_t T)
{
    using namespace sb200;
    clear_error();
    const int rc = wg_check("weight_grad8_workspace", N, O, I, T);
    if (rc) return rc;
    return N == 0 || O == 0 || I == 0 || T == 0 ? 0 : wg_plan(N, O, I, T).bytes;
}

extern "C" int slayer_b200_weight_grad8(float *out, const float *g, const int8_t *q, const uint8_t *scale, int64_t N, int64_t O, int64_t I, int64_t T,
                                        void *workspace, void *stream)
{
    using namespace sb200;
    clear_error();
    const int rc = wg_check("weight_grad8", N, O, I, T);
    if (rc) return rc;
    if (O == 0 || I == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(out, "weight_grad8: null pointer");
    const cudaStream_t st = (cudaStream_t)stream;
    if (N == 0 || T == 0) {
        const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)(O * I) * 4, st);
        if (e != cudaSuccess) { set_error("weight_grad8: %s", cudaGetErrorString(e)); return SLAYER_B200_ECUDA; }
        return SLAYER_B200_OK;
    }
    SB200_REQUIRE(g && q && scale, "weight_grad8: null pointer");
    SB200_REQUIRE(((uintptr_t)out & 3) == 0 && aligned16(g) && aligned16(q), "weight_grad8: a pointer off its alignment");
    SB200_REQUIRE(workspace && aligned16(workspace), "weight_grad8: the workspace must be aligned to 16 bytes");
    int *status = device_status_word();
    if (!status) { set_error("weight_grad8: no status word on this device"); return SLAYER_B200_ECUDA; }
    const WgPlan p = wg_plan(N, O, I, T);
    const int U = (int)ceil_div(T, 16);
    const int inner = (int)std::max<int64_t>(0, N - ceil_div(8, O * T));
    const WgArgs A = {g, q, scale, (float *)workspace, status, N, O, I, T, ceil_div(T, 32), N * O * T, (int)(N * U), (int)p.blocks, U, inner,
                      p.tiles_o, p.tiles * p.blocks, (int)p.shares};
    switch (p.nt) {
    case 256: return wg_align<2, 256>(A, out, p.tiles, st);
    case 128: return wg_align<1, 128>(A, out, p.tiles, st);
    case 64: return wg_align<1, 64>(A, out, p.tiles, st);
    case 32: return wg_align<1, 32>(A, out, p.tiles, st);
    default: return wg_align<1, 16>(A, out, p.tiles, st);
    }
}
