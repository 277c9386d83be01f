// Gated leaky integrator, along the time steps of each row:
//   y_t = f_t y_{t-1} + u_t,   f = sigmoid(gate) or the gate itself,   u = x, or (1 - f) x ("coupled").
// A step is the map h -> A h + B with A = f_t, B = u_t; maps compose to maps, so a row is a scan over them: a lane composes its steps,
// the lanes of a row's group scan their maps with shuffles, and each walks its steps from the state that the lanes before
// it leave.  The backward pass is the same from the other end: c_t = f_t (g_t + c_{t+1}) is what step t hands to step t - 1, and
//   lambda_t = g_t + c_{t+1},   dx = lambda (or (1 - f) lambda),   df = lambda (y_{t-1} - (coupled) x).
// It forms y again from x and the gate, out of the states that the forward pass keeps where each lane begins (4 bytes for 12 or 16 steps), so that
// it reads x, gate and g and writes dx and dgate, and scans once: no y is kept, and none that is rounded to 16 bits is used.  (With states at
// the start of each chunk alone, and a scan for the others, the backward pass took 6 % longer, 64 x 512 x 300, and 14 %, 262144 x 100.)
//
// Maps are floats: A, and 1 - A by itself (R), and B.  A slow leak's f is next to one, where its rounding to 32 bits, taken at each of the thousands of
// steps that such a state remembers, adds up to 1e-4 of it; R has 24 bits of what is forgotten instead.  States are double from chunk to chunk, and
// float within the up to 16 steps that a lane walks.  (All of it in double, with half as many instructions again: 39 + 74 us instead of
// 28 + 49 of the time, 64 x 512 x 300.)  Single steps, and rows of few, are in double throughout.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace sb200 {

constexpr int kLeakThreads = 128;

// CTAs of an SM that registers are rationed for: the most that leave (nearly) none of a lane's steps in memory
template <int K, bool LINED> constexpr int kForwardBlocks = K < 4 ? 9 : LINED ? 7 : 6;
template <int K> constexpr int kBackwardBlocks = K < 4 ? 6 : 5;

template <typename E> __device__ __forceinline__ float to_float(E v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename E> __device__ __forceinline__ E from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// A lane has K vectors of four steps, next to each other; they begin at multiples of four elements of the tensor, not of the row, so that a row's
// first lane may begin with steps of the row before, and vectors are loaded whole whatever T is.  G lanes have a row, or a chunk of it.
constexpr int kVector = 4;

struct LeakShape {
    int rows, T;
    int gate_inner, gate_period;         // gate per row: entry (row / inner) % period; period 0: a gate per step
    int sample_rows;                     // rows with one length
    const int64_t *lengths;              // null: all T
    int chunks;                          // of a row
    int segments, segment_chunks;        // a row's chunks are worked on by `segments` groups of lanes
    bool logit, coupled;
};

struct Row {
    int64_t base;              // first element
    int skew, length;          // elements between the vector it begins in and itself; steps that count
    int reach;                 // elements from its first to the tensor's last, as far as that matters
};

__device__ __forceinline__ Row row_of(const LeakShape &s, int row)
{
    Row r;
    r.base = (int64_t)row * s.T;
    r.skew = (int)(r.base & (kVector - 1));
    r.reach = (int)min((int64_t)(s.rows - row) * s.T, (int64_t)s.T + kVector);
    r.length = s.T;
    if (s.lengths) {
        const int64_t n = __ldg(s.lengths + (unsigned)row / (unsigned)s.sample_rows);
        r.length = n < 0 ? 0 : (n < s.T ? (int)n : s.T);
    }
    return r;
}

template <typename E> struct Packed { using type = uint2; };
template <> struct Packed<float> { using type = uint4; };

// Which of a lane's vectors lie in [0, end) of a row as a whole, and whether one of them lies there in part: its first one, which may begin before the row,
// or the one that `end` is in.  Vectors that begin before `stop` are read whole, though other rows' steps are in them: reach elements from the row's
// first on are the tensor's.  LINED: rows end with their vectors, and all steps count.
// (Without that it is 87 us forward and 153 backward instead of 76 and 147, float32, 78125 x 512.)
template <int K, bool LINED>
struct Inside {
    int t, end, stop;
    bool whole[K], part;
    __device__ __forceinline__ Inside(int t_, int end_, int reach) : t(t_), end(end_), stop(min(end_, reach - 3))
    {
        const int left = end - t;
        part = !LINED && (t < 0 || (left > 0 && left < 4 * K && (left & 3) != 0));
#pragma unroll
        for (int k = 0; k < K; ++k) whole[k] = LINED ? left > 4 * k : (k > 0 || t >= 0) && left >= 4 * k + 4;
    }
};

// Steps [t, t + 4 K) of a row, `fill` where they are outside.  A vector that is there in part is read whole, other rows' steps with it: only
// the tensor's last one may not be.  (One by one it took 2 % longer forward and 16 % backward, float32, 1212121 x 33: 130 and 229 us.)
template <typename E, int K, bool LINED>
__device__ __forceinline__ void load_steps(float (&v)[4 * K], const E *row, const Inside<K, LINED> &in, float fill)
{
    using P = typename Packed<E>::type;
    P raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        E none[4] = {from_float<E>(fill), from_float<E>(fill), from_float<E>(fill), from_float<E>(fill)};
        raw[k] = *reinterpret_cast<P *>(none);
        if (LINED ? in.whole[k] : in.t + 4 * k < in.stop) raw[k] = __ldg(reinterpret_cast<const P *>(row + in.t + 4 * k));
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const E *e = reinterpret_cast<const E *>(&raw[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * k + j] = to_float<E>(e[j]);
    }
    if (in.part) {
#pragma unroll
        for (int j = 0; j < 4 * K; ++j) v[j] = (unsigned)(in.t + j) < (unsigned)in.end ? v[j] : fill;
        if (in.stop < in.end) {     // the tensor's last row
#pragma unroll
            for (int j = 0; j < 4 * K; ++j) {
                const int at = in.t + j;
                if (at >= 0 && at < in.end && in.t + (j & ~3) >= in.stop) v[j] = to_float<E>(row[at]);
            }
        }
    }
}

// results of the steps inside
template <typename E, int K, bool LINED>
__device__ __forceinline__ void store_inside(E *row, const Inside<K, LINED> &in, const float (&v)[4 * K])
{
    using P = typename Packed<E>::type;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        P raw;
        E *e = reinterpret_cast<E *>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = from_float<E>(v[4 * k + j]);
        if (in.whole[k]) *reinterpret_cast<P *>(row + in.t + 4 * k) = raw;
    }
    if (in.part) {
        // the vector that begins before the row, and the one that it ends in
        const int last = (in.end - in.t) >> 2;
        if (in.t < 0) {
#pragma unroll
            for (int j = 1; j < 4; ++j)
                if (in.t + j >= 0 && in.t + j < in.end) row[in.t + j] = from_float<E>(v[j]);
        }
        if (last < K && (last > 0 || in.t >= 0)) {
            float e[3];
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                e[j] = v[j];
#pragma unroll
                for (int k = 1; k < K; ++k) e[j] = last == k ? v[4 * k + j] : e[j];
            }
            const int at = in.t + 4 * last;
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (at + j < in.end) row[at + j] = from_float<E>(e[j]);
        }
    }
}

// and zeros from `in.end` to T
template <typename E, int K, bool LINED>
__device__ __forceinline__ void store_steps(E *row, const Inside<K, LINED> &in, int T, float (&v)[4 * K])
{
    if (LINED || in.end == T) {
        store_inside<E, K, LINED>(row, in, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4 * K; ++j) v[j] = in.t + j < in.end ? v[j] : 0.0f;
        store_inside<E, K, LINED>(row, Inside<K, LINED>(in.t, T, T), v);
    }
}

// f and 1 - f, each to its own 24 bits
struct Decay {
    float f, rest;
};

__device__ __forceinline__ Decay decay_of(float gate, bool logit)
{
    if (!logit) return {gate, 1.0f - gate};
    // e^-|gate| as a power of two, log2(e) in two floats
    float e;
    const float a = fabsf(gate);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-fmaf(a, 1.44269502f, a * 1.92596303e-8f)));
    const float large = __fdividef(1.0f, 1.0f + e), small = e * large;
    return gate < 0.0f ? Decay{small, large} : Decay{1.0f - small, small};
}

// The decay of a whole row.  f = 1 - rest is rounded to 24 bits: taken so at each step, the same part of a rounding would add up over the 16 that a lane
// walks (results 3 to 4 steps of 2^-24 off on average, where it is half of one).  So some steps take the next float above f, and four of
// them forget what they should to an eighth of a rounding each.  A lane of two vectors at most has one f for each, which saves registers
// (8 steps: 62 us backward instead of 69, 3200000 x 8).  With a gate per step the roundings differ from step to step.
struct RowDecay {
    float f[4], rest;
    template <int K> __device__ __forceinline__ Decay at(int j) const { return {f[K < 3 ? j / 4 : j % 4], rest}; }
};

// What a lane knows of its steps.  Those outside of the row, or behind its length, keep the state: f = 1, u = 0.
template <typename E, int K>
struct Steps {
    Decay d[4 * K];
    float x[4 * K];

    template <bool ROW, bool LINED>
    __device__ __forceinline__ void load(const LeakShape &s, const Row &row, const E *x_, const E *gate, const RowDecay &row_d, const Inside<K, LINED> &in)
    {
        load_steps<E, K, LINED>(x, x_ + row.base, in, 0.0f);
        if (!ROW) {
            float g[4 * K];
            load_steps<E, K, LINED>(g, gate + row.base, in, s.logit ? INFINITY : 1.0f);
#pragma unroll
            for (int j = 0; j < 4 * K; ++j) d[j] = decay_of(g[j], s.logit);
        } else {
#pragma unroll
            for (int j = 0; j < 4 * K; ++j) d[j] = in.whole[j / 4] ? row_d.template at<K>(j) : Decay{1.0f, 0.0f};
            if (in.part) {
#pragma unroll
                for (int j = 0; j < 4 * K; ++j)
                    if (in.t + j >= 0 && in.t + j < in.end) d[j] = row_d.template at<K>(j);
            }
        }
    }
    // x is what is added from here on
    __device__ __forceinline__ void couple(bool coupled)
    {
        if (coupled) {
#pragma unroll
            for (int j = 0; j < 4 * K; ++j) x[j] *= d[j].rest;
        }
    }
};

// h -> a h + b, r = 1 - a
struct Map {
    float a, r, b;
    // by what is forgotten of h, or by what is kept: whichever is less
    __device__ __forceinline__ double operator()(double h) const
    {
        const bool little = r < 0.5f;
        return (little ? h : 0.0) + fma((double)(little ? -r : a), h, (double)b);
    }
};

// first, then second
__device__ __forceinline__ Map compose(const Map &first, const Map &second)
{
    const bool little = second.r < 0.5f;
    const float r = fmaf(first.a, second.r, first.r);
    // a product of many factors next to one is off by as many roundings; 1 - r is not
    return {r < 0.5f ? 1.0f - r : first.a * second.a, r, (little ? first.b : 0.0f) + fmaf(little ? -second.r : second.a, first.b, second.b)};
}

// a map, then one step
__device__ __forceinline__ Map step_after(const Map &m, const Decay &d, float u) { return {m.a * d.f, fmaf(m.a, d.rest, m.r), fmaf(d.f, m.b, u)}; }

template <int G>
__device__ __forceinline__ Map shift_up(const Map &m, int d)
{
    return {__shfl_up_sync(~0u, m.a, d, G), __shfl_up_sync(~0u, m.r, d, G), __shfl_up_sync(~0u, m.b, d, G)};
}
template <int G>
__device__ __forceinline__ Map shift_down(const Map &m, int d)
{
    return {__shfl_down_sync(~0u, m.a, d, G), __shfl_down_sync(~0u, m.r, d, G), __shfl_down_sync(~0u, m.b, d, G)};
}
__device__ __forceinline__ Map shift_from(const Map &m, int lane) { return {__shfl_sync(~0u, m.a, lane), __shfl_sync(~0u, m.r, lane), __shfl_sync(~0u, m.b, lane)}; }

// the map of this lane and all before it (FORWARD), or all behind it
template <int G, bool FORWARD>
__device__ __forceinline__ Map scan(Map m, int lane)
{
#pragma unroll
    for (int d = 1; d < G; d *= 2) {
        const Map o = FORWARD ? shift_up<G>(m, d) : shift_down<G>(m, d);
        if (FORWARD ? lane >= d : lane + d < G) m = compose(o, m);
    }
    return m;
}

// the map of the lanes before (behind) this one, from scan()
template <int G, bool FORWARD>
__device__ __forceinline__ Map others(const Map &m, int lane)
{
    if (G == 1) return {1.0f, 0.0f, 0.0f};
    const Map o = FORWARD ? shift_up<G>(m, 1) : shift_down<G>(m, 1);
    return lane == (FORWARD ? 0 : G - 1) ? Map{1.0f, 0.0f, 0.0f} : o;
}

// A state after (FORWARD), or a gradient before, the segments [from, to) of a row; all lanes of a warp get it.  The states of groups of 32 segments
// are double, as those of chunks are.
template <bool FORWARD>
__device__ __forceinline__ double through_segments(const Map *maps, int from, int to, int lane, double h)
{
    for (int at = 0; at < to - from; at += 32) {
        const int k = at + lane;
        Map m = {1.0f, 0.0f, 0.0f};
        if (k < to - from) m = maps[FORWARD ? from + k : to - 1 - k];
        h = shift_from(scan<32, true>(m, lane), 31)(h);
    }
    return h;
}

template <typename E, int K>
__device__ __forceinline__ Map forward_map(const Steps<E, K> &st)
{
    Map m = {st.d[0].f, st.d[0].rest, st.x[0]};
#pragma unroll
    for (int j = 1; j < 4 * K; ++j) m = step_after(m, st.d[j], st.x[j]);
    return m;
}

// c -> f (g + c) for all steps, from the last
template <int N>
__device__ __forceinline__ Map backward_map(const Decay (&d)[N], const float (&g)[N])
{
    Map m = {d[N - 1].f, d[N - 1].rest, d[N - 1].f * g[N - 1]};
#pragma unroll
    for (int j = N - 2; j >= 0; --j) m = {m.a * d[j].f, fmaf(m.a, d[j].rest, m.r), d[j].f * (m.b + g[j])};
    return m;
}

// Which row, segment and lane of its group a thread is; false: none.
template <int G>
__device__ __forceinline__ bool place(const LeakShape &s, int &row, int &segment, int &lane)
{
    const int64_t group = ((int64_t)blockIdx.x * kLeakThreads + threadIdx.x) / G;
    lane = threadIdx.x % G;
    segment = 0;
    if (s.segments > 1) {       // (rows x segments is small then)
        row = (int)((unsigned)group / (unsigned)s.segments);
        segment = (int)group - row * s.segments;
        return row < s.rows;
    }
    row = (int)group;
    return group < s.rows;
}

// (one for a whole row: as exact as 32 bits can be)
__device__ __forceinline__ Decay row_gate(const LeakShape &s, const void *gate, int row)
{
    if (s.gate_period == 0) return {1.0f, 0.0f};
    const float g = __ldg((const float *)gate + (unsigned)row / (unsigned)s.gate_inner % (unsigned)s.gate_period);
    if (!s.logit) return {g, 1.0f - g};
    const float e = expf(-fabsf(g)), small = __fdiv_rn(e, 1.0f + e);
    return g < 0.0f ? Decay{small, 1.0f - small} : Decay{1.0f - small, small};
}

// ROW: kernels of their own for a gate per row (with both kinds in one, its four decays cost a gate per step registers and 4 to 6 %).
template <bool ROW>
__device__ __forceinline__ RowDecay row_gates(const LeakShape &s, const void *gate, int row)
{
    if (!ROW) return {{1.0f, 1.0f, 1.0f, 1.0f}, 0.0f};
    Decay d = row_gate(s, gate, row);
    int up = 0;
    if (s.logit && d.f >= 0.5f) {
        // the float below 1 - rest, and quarters of the way to the next one, 2^-24, that are left (both differences are exact)
        d.f = __fsub_rd(1.0f, d.rest);
        up = __float2int_rn(((1.0f - d.f) - d.rest) * 67108864.0f);
    }
    const float above = __int_as_float(__float_as_int(d.f) + 1);
    return {{up >= 3 ? above : d.f, up >= 1 ? above : d.f, up >= 4 ? above : d.f, up >= 2 ? above : d.f}, d.rest};
}

// Maps one after the other, in double, as states are from chunk to chunk: a segment may have thousands of them, whose sums in float were 130 steps of
// 2^-24 off after 512.
struct Chain {
    double a = 1.0, r = 0.0, b = 0.0;
    __device__ __forceinline__ void add(const Map &m)
    {
        const bool little = m.r < 0.5f;
        r = fma(a, (double)m.r, r);
        a = r < 0.5 ? 1.0 - r : a * (double)m.a;
        b = (little ? b : 0.0) + fma((double)(little ? -m.r : m.a), b, (double)m.b);
    }
};

// Maps of segments: rows too few to fill the GPU are split, and each segment starts from what those before it leave.  ends: what a row's first segment
// (FORWARD), or its last, starts from, in a copy, which the next launch reads: the result that its other end writes may take its place.
template <typename E, int K, bool LINED, bool FORWARD, bool ROW>
__global__ void __launch_bounds__(kLeakThreads)
leak_maps_kernel(Map *maps, float *ends, const E *x, const void *gate, const float *end, const LeakShape s)
{
    int row, segment, lane;
    if (!place<32>(s, row, segment, lane)) return;
    const Row r = row_of(s, row);
    const RowDecay row_d = row_gates<ROW>(s, gate, row);
    Chain all;
    const int first = segment * s.segment_chunks, last = min(first + s.segment_chunks, s.chunks);
    for (int i = first; i < last; ++i) {
        const int c = FORWARD ? i : last - 1 - (i - first);
        Steps<E, K> st;
        st.template load<ROW>(s, r, x, (const E *)gate, row_d, Inside<K, LINED>((c * 32 + lane) * (4 * K) - r.skew, r.length, r.reach));
        if (FORWARD) {
            st.couple(s.coupled);
            all.add(shift_from(scan<32, true>(forward_map<E, K>(st), lane), 31));
        } else {
            all.add(shift_from(scan<32, false>(backward_map<4 * K>(st.d, st.x), lane), 0));
        }
    }
    if (lane == 0) maps[row * s.segments + segment] = {(float)all.a, (float)all.r, (float)all.b};
    if (end && lane == 0 && segment == 0) ends[row] = end[row];
}

template <typename E, int G, int K, bool LINED, bool ROW>
__global__ void __launch_bounds__(kLeakThreads, kForwardBlocks<K, LINED>)
leak_forward_kernel(E *y, float *state, float *starts, const E *x, const void *gate, const float *initial, const Map *maps, const LeakShape s)
{
    int row, segment, lane;
    const bool there = place<G>(s, row, segment, lane);
    if (G == 32 && !there) return;
    if (!there) row = s.rows - 1, segment = 0;      // the shuffles want every lane
    const Row r = row_of(s, row);
    const RowDecay row_d = row_gates<ROW>(s, gate, row);
    double h = initial ? (double)initial[row] : 0.0;
    if (G == 32 && segment > 0) h = through_segments<true>(maps + row * s.segments, 0, segment, lane, h);
    const int first = segment * s.segment_chunks, last = min(first + s.segment_chunks, s.chunks);
    for (int c = first; c < last; ++c) {
        const Inside<K, LINED> in((c * G + lane) * (4 * K) - r.skew, r.length, r.reach);
        Steps<E, K> st;
        st.template load<ROW>(s, r, x, (const E *)gate, row_d, in);
        st.couple(s.coupled);
        const Map m = scan<G, true>(forward_map<E, K>(st), lane);
        float at = (float)others<G, true>(m, lane)(h);
        if (starts && there) starts[((int64_t)row * s.chunks + c) * G + lane] = at;
        h = __shfl_sync(~0u, m(h), G - 1, G);
#pragma unroll
        for (int j = 0; j < 4 * K; ++j) {
            at = fmaf(st.d[j].f, at, st.x[j]);
            st.x[j] = at;
        }
        if (there) store_steps<E, K, LINED>(y + r.base, in, s.T, st.x);
    }
    if (state && there && lane == 0 && segment == s.segments - 1) state[row] = (float)h;
}

// sums: per row and segment, of df: the gradient of a gate per row
template <typename E, int G, int K, bool LINED, bool ROW>
__global__ void __launch_bounds__(kLeakThreads, kBackwardBlocks<K>)
leak_backward_kernel(E *dx, E *dgate, double *sums, float *dinitial, const E *g, const float *gstate, const float *starts, const E *x, const void *gate,
                     const Map *maps, const LeakShape s)
{
    constexpr int N = 4 * K;
    int row, segment, lane;
    const bool there = place<G>(s, row, segment, lane);
    if (G == 32 && !there) return;
    if (!there) row = s.rows - 1, segment = 0;
    const Row r = row_of(s, row);
    const RowDecay row_d = row_gates<ROW>(s, gate, row);
    double carry = gstate ? (double)gstate[row] : 0.0, sum = 0.0;
    if (G == 32 && segment + 1 < s.segments) carry = through_segments<false>(maps + row * s.segments, segment + 1, s.segments, lane, carry);
    const int first = segment * s.segment_chunks, last = min(first + s.segment_chunks, s.chunks);
    for (int c = last - 1; c >= first; --c) {
        const Inside<K, LINED> in((c * G + lane) * N - r.skew, r.length, r.reach);
        float gv[N], slope[N];       // slope: what lambda is multiplied by in dgate
        Steps<E, K> st;
        load_steps<E, K, LINED>(gv, g + r.base, in, 0.0f);
        st.template load<ROW>(s, r, x, (const E *)gate, row_d, in);
        float at = starts[((int64_t)row * s.chunks + c) * G + lane];
#pragma unroll
        for (int j = 0; j < N; ++j) slope[j] = s.coupled ? st.x[j] : 0.0f;
        st.couple(s.coupled);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            slope[j] = at - slope[j];
            if (s.logit) slope[j] *= st.d[j].f * st.d[j].rest;
            at = fmaf(st.d[j].f, at, st.x[j]);
        }
        const Map m = scan<G, false>(backward_map<N>(st.d, gv), lane);
        at = (float)others<G, false>(m, lane)(carry);
        carry = __shfl_sync(~0u, m(carry), 0, G);
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
            const float lambda = gv[j] + at;
            at = st.d[j].f * lambda;
            gv[j] = s.coupled ? lambda * st.d[j].rest : lambda;
            slope[j] *= lambda;
        }
        if (there && dx) store_steps<E, K, LINED>(dx + r.base, in, s.T, gv);
        if (there && dgate) store_steps<E, K, LINED>(dgate + r.base, in, s.T, slope);
        if (sums) {
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) part += (unsigned)(in.t + j) < (unsigned)in.end ? slope[j] : 0.0f;
            sum += (double)part;
        }
    }
    if (sums) {
#pragma unroll
        for (int d = G / 2; d > 0; d /= 2) sum += __shfl_down_sync(~0u, sum, d, G);
        if (there && lane == 0) sums[(int64_t)row * s.segments + segment] = sum;
    }
    if (dinitial && there && lane == 0 && segment == 0) dinitial[row] = (float)carry;
}

// One step of a state in double: by what is forgotten of it, or by what is kept, whichever is less.
__device__ __forceinline__ double step_state(const Decay &d, double h, double u) { return u + (d.f < 0.5f ? (double)d.f * h : fma(-(double)d.rest, h, h)); }

// Rows of up to 13 steps that do not end on vectors, which a lane has alone.  Hardly a vector would be one row's alone, and results would go an element at
// a time (float32: 8000000 x 5 146 us forward and 291 backward, 3000000 x 13 115 and 200; so it is 112 and 206, 77 and 168).  A CTA's rows are one piece of memory that begins at 16 bytes: it is copied to
// shared memory as it is, a thread walks a row there, its state in double, and results go back the same way.
constexpr int kShortSteps = 13;

template <typename E>
__device__ __forceinline__ void short_fetch(E *tile, const E *from, int count)
{
    constexpr int W = 16 / (int)sizeof(E);
    const int whole = count / W;
    for (int i = threadIdx.x; i < whole; i += kLeakThreads)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(tile + i * W)), "l"(from + i * W) : "memory");
    for (int i = whole * W + threadIdx.x; i < count; i += kLeakThreads) tile[i] = from[i];
}

__device__ __forceinline__ void short_fetched()
{
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}

template <typename E>
__device__ __forceinline__ void short_store(E *to, const E *tile, int count)
{
    constexpr int W = 16 / (int)sizeof(E);
    const int whole = count / W;
    for (int i = threadIdx.x; i < whole; i += kLeakThreads) reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(tile)[i];
    for (int i = whole * W + threadIdx.x; i < count; i += kLeakThreads) to[i] = tile[i];
}

template <typename E>
__global__ void __launch_bounds__(kLeakThreads)
leak_short_forward_kernel(E *y, float *state, float *starts, const E *x, const void *gate, const float *initial, const LeakShape s)
{
    extern __shared__ __align__(16) unsigned char short_memory[];
    E *const xs = reinterpret_cast<E *>(short_memory), *const gs = xs + kLeakThreads * s.T;
    const int64_t first = (int64_t)blockIdx.x * kLeakThreads;
    const int here = (int)min((int64_t)kLeakThreads, s.rows - first), count = here * s.T;
    short_fetch(xs, x + first * s.T, count);
    if (s.gate_period == 0) short_fetch(gs, (const E *)gate + first * s.T, count);
    short_fetched();
    if (threadIdx.x < here) {
        const int row = (int)first + threadIdx.x, length = row_of(s, row).length;
        const Decay row_d = row_gate(s, gate, row);
        E *const xr = xs + threadIdx.x * s.T;
        const E *const gr = gs + threadIdx.x * s.T;
        double h = initial ? (double)initial[row] : 0.0;
        if (starts) starts[row] = (float)h;
        for (int t = 0; t < s.T; ++t) {
            if (t < length) {
                const Decay d = s.gate_period ? row_d : decay_of(to_float<E>(gr[t]), s.logit);
                const float v = to_float<E>(xr[t]);
                h = step_state(d, h, (double)(s.coupled ? d.rest * v : v));
            }
            xr[t] = from_float<E>(t < length ? (float)h : 0.0f);
        }
        if (state) state[row] = (float)h;
    }
    __syncthreads();
    short_store(y + first * s.T, xs, count);
}

template <typename E>
__global__ void __launch_bounds__(kLeakThreads)
leak_short_backward_kernel(E *dx, E *dgate, double *sums, float *dinitial, const E *g, const float *gstate, const float *starts, const E *x, const void *gate,
                           const LeakShape s)
{
    extern __shared__ __align__(16) unsigned char short_memory[];
    E *const xs = reinterpret_cast<E *>(short_memory), *const gs = xs + kLeakThreads * s.T, *const up = gs + kLeakThreads * s.T;
    float *const slopes = reinterpret_cast<float *>(up + kLeakThreads * s.T);        // what lambda is multiplied by in dgate
    const int64_t first = (int64_t)blockIdx.x * kLeakThreads;
    const int here = (int)min((int64_t)kLeakThreads, s.rows - first), count = here * s.T;
    short_fetch(xs, x + first * s.T, count);
    short_fetch(up, g + first * s.T, count);
    if (s.gate_period == 0) short_fetch(gs, (const E *)gate + first * s.T, count);
    short_fetched();
    if (threadIdx.x < here) {
        const int row = (int)first + threadIdx.x, length = row_of(s, row).length;
        const Decay row_d = row_gate(s, gate, row);
        E *const xr = xs + threadIdx.x * s.T, *const gr = gs + threadIdx.x * s.T;
        const E *const ur = up + threadIdx.x * s.T;
        float *const slope = slopes + threadIdx.x * s.T;
        double at = starts[row], sum = 0.0;
        for (int t = 0; t < length; ++t) {
            const Decay d = s.gate_period ? row_d : decay_of(to_float<E>(gr[t]), s.logit);
            const float v = to_float<E>(xr[t]), k = (float)at - (s.coupled ? v : 0.0f);
            slope[t] = s.logit ? k * (d.f * d.rest) : k;
            at = step_state(d, at, (double)(s.coupled ? d.rest * v : v));
        }
        double carry = gstate ? (double)gstate[row] : 0.0;
        for (int t = s.T - 1; t >= 0; --t) {
            float to_x = 0.0f, to_gate = 0.0f;
            if (t < length) {
                const Decay d = s.gate_period ? row_d : decay_of(to_float<E>(gr[t]), s.logit);
                const double lambda = (double)to_float<E>(ur[t]) + carry;
                carry = step_state(d, lambda, 0.0);
                to_x = s.coupled ? (float)lambda * d.rest : (float)lambda;
                to_gate = (float)lambda * slope[t];
                sum += (double)to_gate;
            }
            xr[t] = from_float<E>(to_x);
            if (dgate) gr[t] = from_float<E>(to_gate);
        }
        if (sums) sums[row] = sum;
        if (dinitial) dinitial[row] = (float)carry;
    }
    __syncthreads();
    if (dx) short_store(dx + first * s.T, xs, count);
    if (dgate) short_store(dgate + first * s.T, gs, count);
}

// The gradient of a gate per row is the sum over the rows that have it, in a fixed order: rows (k period + i) inner + j of gate i.  By the number of them:
// up to 16, a thread a gate; up to 512, eight warps for 32 gates, whose entries lie next to each other where inner is 1, or a warp a gate where inner is
// 16 or more; else, and where all gates' CTAs are resident at once, a CTA a gate.  (A CTA for each of 8000000 gates of one row took 12370 us beside a
// backward pass of 152, threads take 32; 9248 gates of 32 rows 19.2 and 4.4.  1000 gates of 500 rows: CTAs 5.4, warps 9.5.)
__device__ __forceinline__ int64_t gate_entry(unsigned n, unsigned inner, int64_t period, int64_t i) { return ((int64_t)(n / inner) * period + i) * inner + n % inner; }

// P warps have 32 gates
template <int P>
__global__ void __launch_bounds__(256)
leak_gates_sum_kernel(float *out, const double *sums, unsigned count, int64_t period, unsigned inner)
{
    __shared__ double part[P > 1 ? 8 : 1][32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, p = warp % P;
    const int64_t i = ((int64_t)blockIdx.x * (8 / P) + warp / P) * 32 + lane;
    double sum = 0.0;
    if (i < period) {
#pragma unroll 8
        for (unsigned n = p; n < count; n += P) sum += sums[gate_entry(n, inner, period, i)];
    }
    if (P > 1) {
        part[warp][lane] = sum;
        __syncthreads();
        if (p > 0) return;
#pragma unroll
        for (int w = 1; w < P; ++w) sum += part[warp + w][lane];
    }
    if (i < period) out[i] = (float)sum;
}

__global__ void __launch_bounds__(256)
leak_gate_warp_sum_kernel(float *out, const double *sums, unsigned count, int64_t period, unsigned inner)
{
    const int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
    if (i >= period) return;
    double sum = 0.0;
#pragma unroll 4
    for (unsigned n = threadIdx.x % 32; n < count; n += 32) sum += sums[gate_entry(n, inner, period, i)];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_down_sync(~0u, sum, d);
    if (threadIdx.x % 32 == 0) out[i] = (float)sum;
}

// A CTA.  parts > 1: each of them sums every parts-th entry, and a second launch (inner = parts, period = gates, outer = 1) those.
__global__ void __launch_bounds__(256)
leak_gate_sum_kernel(double *part, float *out, const double *sums, int64_t outer, int64_t period, int64_t inner, int64_t parts)
{
    __shared__ double warp_sum[8];
    const int64_t i = blockIdx.x / parts, p = blockIdx.x % parts, count = outer * inner;
    double sum = 0.0;
    for (int64_t n = p * 256 + threadIdx.x; n < count; n += parts * 256) sum += sums[(n / inner * period + i) * inner + n % inner];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_down_sync(~0u, sum, d);
    if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    sum = 0.0;
    for (int w = 0; w < 8; ++w) sum += warp_sum[w];
    if (part) part[blockIdx.x] = sum;
    else out[i] = (float)sum;
}

// one time step: state and output of each row
template <typename E, typename EG>
__global__ void __launch_bounds__(256)
leak_step_kernel(E *y, float *state, const E *x, const EG *gate, int64_t rows, int64_t inner, int64_t period, bool logit, bool coupled)
{
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= rows) return;
    const Decay d = decay_of(to_float<EG>(gate[period ? row / inner % period : row]), logit);
    const float v = to_float<E>(x[row]);
    const float h = (float)step_state(d, (double)state[row], (double)(coupled ? d.rest * v : v));
    state[row] = h;
    y[row] = from_float<E>(h);
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int64_t kGateCount = 8192;      // entries that one CTA adds up

// Lanes of a row and vectors of a lane.  Rows of up to 512 steps have as few lanes as hold them, with three or four vectors each (two maps of 16 bytes are
// passed on in each doubling of the lanes, whatever a lane holds); longer ones are worked on in chunks of 32 lanes with four.
struct LeakLanes {
    int lanes, vectors;
};

static LeakLanes lanes_of(int64_t T)
{
    const int64_t n = ceil_div(T + (T % kVector ? kVector - 1 : 0), kVector);
    if (n <= 1) return {1, 1};
    if (n <= 2) return {1, 2};
    if (n <= 4) return {1, 4};
    for (int g = 2; g <= 32; g *= 2) {
        if (n <= 3 * g) return {g, 3};
        if (n <= 4 * g) return {g, 4};
    }
    return {32, 4};
}

static int64_t chunks_of(int64_t T)
{
    const LeakLanes l = lanes_of(T);
    return ceil_div(T + (T % kVector ? kVector - 1 : 0), (int64_t)l.lanes * l.vectors * kVector);
}

// groups per row: rows with many chunks, too few to give every SM 16 warps, are split.
static int64_t segments_of(int64_t rows, int64_t T)
{
    const int64_t chunks = chunks_of(T), warps = (int64_t)sm_count() * 16;
    if (chunks < 2 || rows * 2 > warps) return 1;
    int64_t n = warps / rows;
    if (n > chunks) n = chunks;
    if (n > 1024) n = 1024;
    return ceil_div(chunks, ceil_div(chunks, n));
}

static bool known(int dtype) { return dtype == SLAYER_B200_F32 || dtype == SLAYER_B200_BF16 || dtype == SLAYER_B200_F16; }

struct LeakPlan {
    LeakShape s;
    LeakLanes l;
    bool lined;                          // rows end with their vectors, and all of their steps count
    int64_t ends_at, maps_bytes, sums_bytes, gate_parts;         // (maps_bytes: with ends)
};

static int plan_leak(LeakPlan &p, const char *op, int dtype, int flags, int64_t rows, int64_t T, const int64_t *lengths, int64_t sample_rows,
                     int64_t gate_inner, int64_t gate_period)
{
    SB200_REQUIRE(known(dtype), "%s: unknown element type %d", op, dtype);
    SB200_REQUIRE((flags & ~3) == 0, "%s: unknown flags %d", op, flags);
    SB200_REQUIRE(rows >= 0 && T >= 0, "%s: negative size", op);
    SB200_REQUIRE(rows <= ((int64_t)1 << 31) - 64 && T <= (int64_t)1 << 30, "%s: at most 2^31 - 64 rows of 2^30 steps", op);
    SB200_REQUIRE(gate_period >= 0 && (gate_period == 0 || gate_inner >= 1), "%s: bad gate layout", op);
    SB200_REQUIRE(gate_period == 0 || (gate_period <= rows && gate_inner <= rows && rows % (gate_inner * gate_period) == 0) || rows == 0,
                  "%s: rows must be whole groups of gates", op);
    SB200_REQUIRE(!lengths || sample_rows >= 1, "%s: lengths need the number of rows that have one", op);
    p.l = lanes_of(T);
    p.lined = T % kVector == 0 && !lengths;
    const int64_t chunks = chunks_of(T), segments = rows ? segments_of(rows, T) : 1;
    p.s = {(int)rows, (int)T, (int)gate_inner, (int)gate_period, (int)(sample_rows < rows ? sample_rows : rows), lengths, (int)chunks, (int)segments,
           (int)ceil_div(chunks, segments), (flags & SLAYER_B200_LEAK_LOGIT) != 0, (flags & SLAYER_B200_LEAK_COUPLED) != 0};
    p.ends_at = ceil_div(rows * segments * (int64_t)sizeof(Map), 16) * 16;
    p.maps_bytes = segments > 1 ? p.ends_at + ceil_div(rows * (int64_t)sizeof(float), 16) * 16 : 0;
    p.sums_bytes = p.gate_parts = 0;
    if (gate_period && rows) {
        const int64_t count = rows / gate_period * segments;
        p.gate_parts = ceil_div(count, kGateCount);
        if (p.gate_parts > 1024) p.gate_parts = 1024;
        p.sums_bytes = (rows * segments + (p.gate_parts > 1 ? gate_period * p.gate_parts : 0)) * (int64_t)sizeof(double);
    }
    SB200_REQUIRE(ceil_div(rows * segments * p.l.lanes, kLeakThreads) <= 0x7fffffff, "%s: too many rows", op);
    SB200_REQUIRE(p.gate_parts * gate_period <= 0x7fffffff, "%s: too many gates", op);
    return SLAYER_B200_OK;
}

template <typename E, int G, int K, bool LINED, bool ROW>
static void run_forward(const LeakPlan &p, void *y, float *state, float *starts, const void *x, const void *gate, const float *initial, void *workspace,
                        cudaStream_t st)
{
    Map *maps = (Map *)workspace;
    const unsigned blocks = (unsigned)ceil_div((int64_t)p.s.rows * p.s.segments * G, kLeakThreads);
    if constexpr (G == 32)
        if (p.s.segments > 1) {
            float *const ends = (float *)((char *)workspace + p.ends_at);
            leak_maps_kernel<E, K, LINED, true, ROW><<<blocks, kLeakThreads, 0, st>>>(maps, ends, (const E *)x, gate, initial, p.s);
            if (initial) initial = ends;
        }
    if constexpr (G == 1 && !LINED)
        if (p.s.T % kVector != 0 && p.s.T <= kShortSteps) {
            leak_short_forward_kernel<E><<<blocks, kLeakThreads, 2 * kLeakThreads * p.s.T * sizeof(E), st>>>((E *)y, state, starts, (const E *)x, gate, initial,
                                                                                                            p.s);
            return;
        }
    leak_forward_kernel<E, G, K, LINED, ROW><<<blocks, kLeakThreads, 0, st>>>((E *)y, state, starts, (const E *)x, gate, initial, maps, p.s);
}

static void sum_gates(float *out, const double *sums, int64_t outer, int64_t period, int64_t inner, cudaStream_t st)
{
    const int64_t count = outer * inner;
    const bool one_wave = period <= (int64_t)sm_count() * 8;
    if (count > 512 || (count > 16 && one_wave)) leak_gate_sum_kernel<<<(unsigned)period, 256, 0, st>>>(nullptr, out, sums, outer, period, inner, 1);
    else if (count <= 16) leak_gates_sum_kernel<1><<<(unsigned)ceil_div(period, 256), 256, 0, st>>>(out, sums, (unsigned)count, period, (unsigned)inner);
    else if (inner >= 16) leak_gate_warp_sum_kernel<<<(unsigned)ceil_div(period, 8), 256, 0, st>>>(out, sums, (unsigned)count, period, (unsigned)inner);
    else leak_gates_sum_kernel<8><<<(unsigned)ceil_div(period, 32), 256, 0, st>>>(out, sums, (unsigned)count, period, (unsigned)inner);
}

template <typename E, int G, int K, bool LINED, bool ROW>
static void run_backward(const LeakPlan &p, void *dx, void *dgate, float *dinitial, const void *g, const float *gstate, const float *starts, const void *x,
                         const void *gate, void *workspace, cudaStream_t st)
{
    Map *maps = (Map *)workspace;
    double *sums = (double *)((char *)workspace + p.maps_bytes);
    const bool per_row = p.s.gate_period > 0;
    const unsigned blocks = (unsigned)ceil_div((int64_t)p.s.rows * p.s.segments * G, kLeakThreads);
    if constexpr (G == 32)
        if (p.s.segments > 1) {
            float *const ends = (float *)((char *)workspace + p.ends_at);
            leak_maps_kernel<E, K, LINED, false, ROW><<<blocks, kLeakThreads, 0, st>>>(maps, ends, (const E *)g, gate, gstate, p.s);
            if (gstate) gstate = ends;
        }
    E *const to_gate = per_row ? nullptr : (E *)dgate;
    double *const to_sums = per_row && dgate ? sums : nullptr;
    bool done = false;
    if constexpr (G == 1 && !LINED)
        if (p.s.T % kVector != 0 && p.s.T <= kShortSteps) {
            leak_short_backward_kernel<E><<<blocks, kLeakThreads, kLeakThreads * p.s.T * (3 * sizeof(E) + sizeof(float)), st>>>(
                (E *)dx, to_gate, to_sums, dinitial, (const E *)g, gstate, starts, (const E *)x, gate, p.s);
            done = true;
        }
    if (!done)
        leak_backward_kernel<E, G, K, LINED, ROW><<<blocks, kLeakThreads, 0, st>>>((E *)dx, to_gate, to_sums, dinitial, (const E *)g, gstate, starts,
                                                                                   (const E *)x, gate, maps, p.s);
    if (per_row && dgate) {
        const int64_t inner = (int64_t)p.s.gate_inner * p.s.segments, outer = p.s.rows / ((int64_t)p.s.gate_inner * p.s.gate_period);
        double *part = sums + (int64_t)p.s.rows * p.s.segments;
        if (p.gate_parts > 1) {
            leak_gate_sum_kernel<<<(unsigned)(p.s.gate_period * p.gate_parts), 256, 0, st>>>(part, nullptr, sums, outer, p.s.gate_period, inner, p.gate_parts);
            sum_gates((float *)dgate, part, 1, p.s.gate_period, p.gate_parts, st);
        } else {
            sum_gates((float *)dgate, sums, outer, p.s.gate_period, inner, st);
        }
    }
}

// the kernel of a plan's lanes and vectors
#define SB200_LEAK_LANES(E, CALL)                                                              \
    switch (p.l.lanes) {                                                                       \
    case 1: if (p.l.vectors == 1) CALL(E, 1, 1); else if (p.l.vectors == 2) CALL(E, 1, 2); else CALL(E, 1, 4); break; \
    case 2: if (p.l.vectors == 3) CALL(E, 2, 3); else CALL(E, 2, 4); break;                    \
    case 4: if (p.l.vectors == 3) CALL(E, 4, 3); else CALL(E, 4, 4); break;                    \
    case 8: if (p.l.vectors == 3) CALL(E, 8, 3); else CALL(E, 8, 4); break;                    \
    case 16: if (p.l.vectors == 3) CALL(E, 16, 3); else CALL(E, 16, 4); break;                 \
    default: if (p.l.vectors == 3) CALL(E, 32, 3); else CALL(E, 32, 4); break;                 \
    }
#define SB200_LEAK_TYPES(CALL)                                                \
    if (dtype == SLAYER_B200_F32) { SB200_LEAK_LANES(float, CALL) }           \
    else if (dtype == SLAYER_B200_BF16) { SB200_LEAK_LANES(__nv_bfloat16, CALL) } \
    else { SB200_LEAK_LANES(__half, CALL) }

static bool element_aligned(const void *p, int dtype) { return ((uintptr_t)p & (dtype == SLAYER_B200_F32 ? 3 : 1)) == 0; }
static bool aligned_to(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

struct Memory {
    const void *p;
    int64_t bytes;
};

static bool apart(const Memory &a, const Memory &b)
{
    return !a.p || !b.p || (uintptr_t)a.p + (uintptr_t)a.bytes <= (uintptr_t)b.p || (uintptr_t)b.p + (uintptr_t)b.bytes <= (uintptr_t)a.p;
}

// What is written shares nothing with the rest: groups of lanes read what others would have written.  list: the first `written` of it are; `end` of those may
// be `start` of the others.
template <int N>
static bool all_apart(const Memory (&list)[N], int written, int end, int start)
{
    for (int i = 0; i < written; ++i)
        for (int j = i + 1; j < N; ++j)
            if (!apart(list[i], list[j]) && !(i == end && j == start && list[i].p == list[j].p)) return false;
    return true;
}

static int64_t gate_bytes(const LeakPlan &p, int64_t element) { return p.s.gate_period ? p.s.gate_period * (int64_t)sizeof(float) : (int64_t)p.s.rows * p.s.T * element; }
static int64_t lengths_bytes(const LeakPlan &p) { return p.s.lengths ? ceil_div(p.s.rows, p.s.sample_rows) * (int64_t)sizeof(int64_t) : 0; }

}  // namespace sb200

extern "C" int64_t slayer_b200_leak_states(int64_t T)
{
    using namespace sb200;
    clear_error();
    SB200_REQUIRE(T >= 0 && T <= (int64_t)1 << 30, "leak_states: bad length");
    return chunks_of(T) * lanes_of(T).lanes;
}

extern "C" int64_t slayer_b200_leak_workspace(int64_t rows, int64_t T, int dtype, int64_t gate_inner, int64_t gate_period)
{
    using namespace sb200;
    clear_error();
    LeakPlan p;
    const int rc = plan_leak(p, "leak_workspace", dtype, 0, rows, T, nullptr, 1, gate_inner, gate_period);
    return rc ? rc : p.maps_bytes + p.sums_bytes;
}

extern "C" int slayer_b200_leak_forward(void *y, float *state, float *starts, const void *x, const void *gate, const float *initial, int dtype, int flags,
                                        int64_t rows, int64_t T, const int64_t *lengths, int64_t sample_rows, int64_t gate_inner, int64_t gate_period,
                                        void *workspace, void *stream)
{
    using namespace sb200;
    clear_error();
    LeakPlan p;
    const int rc = plan_leak(p, "leak_forward", dtype, flags, rows, T, lengths, sample_rows, gate_inner, gate_period);
    if (rc) return rc;
    if (rows == 0) return SLAYER_B200_OK;
    SB200_REQUIRE((y && x) || T == 0, "leak_forward: null pointer");
    SB200_REQUIRE(gate || (T == 0 && gate_period == 0), "leak_forward: null pointer");
    SB200_REQUIRE(p.maps_bytes == 0 || (workspace && aligned16(workspace)), "leak_forward: the workspace must be aligned to 16 bytes");
    SB200_REQUIRE(aligned16(y) && aligned16(x) && aligned_to(gate, gate_period ? 4 : 16) && aligned_to(state, 4) && aligned_to(starts, 4) &&
                      aligned_to(initial, 4) && aligned_to(lengths, 8),
                  "leak_forward: a pointer off its alignment");
    const int64_t element = dtype == SLAYER_B200_F32 ? 4 : 2, all = rows * T * element, per_row = rows * (int64_t)sizeof(float);
    const Memory list[] = {{y, all}, {state, per_row}, {starts, per_row * p.s.chunks * p.l.lanes}, {workspace, p.maps_bytes},
                           {x, all}, {gate, gate_bytes(p, element)}, {initial, per_row}, {lengths, lengths_bytes(p)}};
    SB200_REQUIRE(all_apart(list, 4, 1, 6), "leak_forward: y, state, starts and the workspace share memory with one another or with what is read");
    const cudaStream_t st = (cudaStream_t)stream;
#define SB200_LEAK_CALL(E, G, K)                                                                          \
    do {                                                                                                  \
        const auto run = p.s.gate_period ? p.lined ? run_forward<E, G, K, true, true> : run_forward<E, G, K, false, true>    \
                                         : p.lined ? run_forward<E, G, K, true, false> : run_forward<E, G, K, false, false>; \
        run(p, y, state, starts, x, gate, initial, workspace, st);                                        \
    } while (0)
    SB200_LEAK_TYPES(SB200_LEAK_CALL)
#undef SB200_LEAK_CALL
    return check_launch("leak_forward kernel launch");
}

extern "C" int slayer_b200_leak_backward(void *dx, void *dgate, float *dinitial, const void *g, const float *gstate, const float *starts, const void *x,
                                         const void *gate, int dtype, int flags, int64_t rows, int64_t T, const int64_t *lengths, int64_t sample_rows,
                                         int64_t gate_inner, int64_t gate_period, void *workspace, void *stream)
{
    using namespace sb200;
    clear_error();
    LeakPlan p;
    const int rc = plan_leak(p, "leak_backward", dtype, flags, rows, T, lengths, sample_rows, gate_inner, gate_period);
    if (rc) return rc;
    if (rows == 0) return SLAYER_B200_OK;
    SB200_REQUIRE((g && x && starts) || T == 0, "leak_backward: null pointer");
    SB200_REQUIRE(gate || (T == 0 && gate_period == 0), "leak_backward: null pointer");
    SB200_REQUIRE(p.maps_bytes + p.sums_bytes == 0 || (workspace && aligned16(workspace)), "leak_backward: the workspace must be aligned to 16 bytes");
    SB200_REQUIRE(aligned16(dx) && aligned_to(dgate, gate_period ? 4 : 16) && aligned16(g) && aligned16(x) && aligned_to(gate, gate_period ? 4 : 16) &&
                      aligned_to(dinitial, 4) && aligned_to(gstate, 4) && aligned_to(starts, 4) && aligned_to(lengths, 8),
                  "leak_backward: a pointer off its alignment");
    const int64_t element = dtype == SLAYER_B200_F32 ? 4 : 2, all = rows * T * element, per_row = rows * (int64_t)sizeof(float);
    const Memory list[] = {{dx, all}, {dgate, gate_bytes(p, element)}, {dinitial, per_row}, {workspace, p.maps_bytes + p.sums_bytes},
                           {g, all}, {gstate, per_row}, {starts, per_row * p.s.chunks * p.l.lanes}, {x, all}, {gate, gate_bytes(p, element)},
                           {lengths, lengths_bytes(p)}};
    SB200_REQUIRE(all_apart(list, 4, 2, 5), "leak_backward: dx, dgate, dinitial and the workspace share memory with one another or with what is read");
    const cudaStream_t st = (cudaStream_t)stream;
#define SB200_LEAK_CALL(E, G, K)                                                                          \
    do {                                                                                                  \
        const auto run = p.s.gate_period ? p.lined ? run_backward<E, G, K, true, true> : run_backward<E, G, K, false, true>    \
                                         : p.lined ? run_backward<E, G, K, true, false> : run_backward<E, G, K, false, false>; \
        run(p, dx, dgate, dinitial, g, gstate, starts, x, gate, workspace, st);                           \
    } while (0)
    SB200_LEAK_TYPES(SB200_LEAK_CALL)
#undef SB200_LEAK_CALL
    return check_launch("leak_backward kernel launch");
}

extern "C" int slayer_b200_leak_step(void *y, float *state, const void *x, const void *gate, int dtype, int gate_dtype, int flags, int64_t rows,
                                     int64_t gate_inner, int64_t gate_period, void *stream)
{
    using namespace sb200;
    clear_error();
    LeakPlan p;
    const int rc = plan_leak(p, "leak_step", dtype, flags, rows, 1, nullptr, 1, gate_inner, gate_period);
    if (rc) return rc;
    SB200_REQUIRE(gate_dtype == dtype || gate_dtype == SLAYER_B200_F32, "leak_step: the gate has x's type or float32");
    if (rows == 0) return SLAYER_B200_OK;
    SB200_REQUIRE(y && state && x && gate, "leak_step: null pointer");
    SB200_REQUIRE(element_aligned(y, dtype) && element_aligned(x, dtype) && element_aligned(gate, gate_dtype) && aligned_to(state, 4),
                  "leak_step: a pointer off its element's alignment");
    const int64_t element = dtype == SLAYER_B200_F32 ? 4 : 2, gates = (gate_period ? gate_period : rows) * (gate_dtype == SLAYER_B200_F32 ? 4 : 2);
    const Memory out = {y, rows * element}, kept = {state, rows * 4}, in = {x, rows * element}, by = {gate, gates};
    SB200_REQUIRE(apart(kept, out) && apart(kept, in) && apart(kept, by), "leak_step: state shares memory with y, x or gate");
    // (a thread reads its own elements of the two before it writes its own of y)
    SB200_REQUIRE((apart(out, in) || y == x) && (apart(out, by) || (y == gate && gate_period == 0 && gate_dtype == dtype)),
                  "leak_step: y shares memory with other elements of x or gate");
    const unsigned blocks = (unsigned)ceil_div(rows, 256);
    const cudaStream_t st = (cudaStream_t)stream;
#define SB200_LEAK_STEP(E, EG)                                                                                                                       \
    leak_step_kernel<E, EG><<<blocks, 256, 0, st>>>((E *)y, state, (const E *)x, (const EG *)gate, rows, gate_inner, gate_period, p.s.logit, p.s.coupled)
    if (dtype == SLAYER_B200_F32) SB200_LEAK_STEP(float, float);
    else if (dtype == SLAYER_B200_BF16 && gate_dtype == SLAYER_B200_F32) SB200_LEAK_STEP(__nv_bfloat16, float);
    else if (dtype == SLAYER_B200_BF16) SB200_LEAK_STEP(__nv_bfloat16, __nv_bfloat16);
    else if (gate_dtype == SLAYER_B200_F32) SB200_LEAK_STEP(__half, float);
    else SB200_LEAK_STEP(__half, __half);
#undef SB200_LEAK_STEP
    return check_launch("leak_step kernel launch");
}
