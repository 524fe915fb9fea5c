// Layer norm (include/aetcnn_ops.h): forward, and backward with the reduction of
// the scales' and biases' gradients.
//
// Bound by memory.  A row of up to 4096 chunks of 16 bytes (backward, 16-bit
// types: 2048) lies in the registers of the G threads that share it, I chunks each,
// so that it is read once: its sums, then its values.  Short rows share a wave, rows of
// more than a few thousand values take a workgroup of 256 to 1024 threads.
// Workgroups run over rows and keep the parameters, and in the backward pass the
// sums of the parameters' gradients, in registers; the next row is loaded while
// one is worked on.  Longer rows are cut into parts, in two passes over memory.
#include "checkpoint.hpp"

#include <math.h>

namespace ach {
namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));

// ---- sums over the G threads of a row; every thread gets them -------------------
template <int CTRL> __device__ __forceinline__ float moved(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ double moved(double v)
{
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true),
                   hi = __builtin_amdgcn_mov_dpp((int)(u >> 32), CTRL, 0xf, 0xf, true);
    return __longlong_as_double((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float of_lane(float v, int lane) { return lane_value(v, lane); }
__device__ __forceinline__ double of_lane(double v, int lane)
{
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane),
                   hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __longlong_as_double((uint64_t)hi << 32 | lo);
}
// Within 16 lanes by their mirror images, over a wave by its four sixteens, over a
// workgroup through `sh`, which holds N values per wave and must not have been read
// since the last barrier but one.
template <int G, int N, class V> __device__ __forceinline__ void row_sums(V *v, V *sh)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] += moved<0xb1>(v[i]);
        v[i] += moved<0x4e>(v[i]);
        v[i] += moved<0x141>(v[i]);
        v[i] += moved<0x140>(v[i]);
        if (G >= 64) v[i] = of_lane(v[i], 0) + of_lane(v[i], 16) + of_lane(v[i], 32) + of_lane(v[i], 48);
    }
    if (G <= 64) return;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) sh[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sh[i];
#pragma unroll
    for (int w = 1; w < G / 64; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += sh[w * N + i];
}

// Values into y or dx.  What the L2 caches (8 of 4 MB) do not hold beside the rows that
// are read, as much again, is stored past the caches, where it would take the place of
// rows that are still to be read (4096 x 8192 bf16 forward: 32 us, 23 past them; 128 x
// 186624 fp32, which is read twice: 66 and 55; backward 2048 x 4000 fp32, 33 MB, 29 and
// 23, 1100 x 4000, 18 MB, 16.6 and 16.4, forward 9.1 and 7.9).
template <int TYPE>
__device__ __forceinline__ void write_values(typename Elem<TYPE>::T *p, int left, const float *v, bool past)
{
    if (past) store_values<TYPE, true>(p, left, v);
    else store_values<TYPE>(p, left, v);
}

// ---- chunks ------------------------------------------------------------------------
// 16 bytes as they lie in memory, of which `left` values are there (the others: fill).
template <int TYPE>
__device__ __forceinline__ v4u load_chunk(const typename Elem<TYPE>::T *p, int left, float fill)
{
    constexpr int VEC = Row<TYPE>::VEC;
    using T = typename Elem<TYPE>::T;
    if (left >= VEC) {
        const typename Row<TYPE>::Chunk c = Row<TYPE>::load(p);
        return __builtin_bit_cast(v4u, c);
    }
    typename Row<TYPE>::Chunk c;
#pragma unroll
    for (int i = 0; i < VEC; ++i) c[i] = (T)fill;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (i < left) c[i] = p[i];
    return __builtin_bit_cast(v4u, c);
}
template <int TYPE> __device__ __forceinline__ void chunk_values(v4u c, float *v)
{
    const typename Row<TYPE>::Chunk t = __builtin_bit_cast(typename Row<TYPE>::Chunk, c);
#pragma unroll
    for (int i = 0; i < Row<TYPE>::VEC; ++i) v[i] = (float)t[i];
}

// Keeps the compiler from holding a chunk's values, twice the registers, from one
// use of it to the next.
__device__ __forceinline__ void forget(v4u &c)
{
    asm volatile("" : "+v"(c));
}

// ---- forward -------------------------------------------------------------------------
struct Fwd {
    bool past;                   // y past the caches
    int rows, features, chunks;  // chunks of a row: with a checkpoint, of whole blocks
    double inv;                  // 1 / features
    float eps;
    int64_t stride, y_stride;
    const float *scales, *biases;
    float *stats;
    Kept k;
    double2 *part;   // of rows in parts: [rows][parts] sums,
    float *first;    // [rows] first values
    int parts, span; // chunks of a part
};

// From the sums of x - first and of their squares, differences and sums in 64 bits:
// where the first value is far from the others, these differences would all round
// alike in 32, and the mean move by as much (186624 values of 0.3 behind one of 1000:
// by 4e-5 of itself).  As the row's first value is one of its n, the mean is at most
// sqrt(n) deviations from it, and the subtraction of its square loses log2 n of the 53
// bits at most.  (The variance passes a float's range where the values pass 1.8e19.)
__device__ __forceinline__ float2 statistics(double s, double q, float first, double inv, float eps)
{
    const double m = s * inv, var = fmax(q * inv - m * m, 0.) + (double)eps;
    const float v = (float)var, mean = (float)((double)first + m);
    float r;
    if (v < 0x1p120f) {
        r = __builtin_amdgcn_rsqf(v);
        r = fmaf(.5f * r, fmaf(-v * r, r, 1.f), r);
    } else {
        r = (float)(1. / sqrt(var));
    }
    return make_float2(mean, q < (double)INFINITY ? r : NAN);
}

// x_norm from a row's mean and rstd, in halves: x - mean may pass a float's range
// where neither does (both factors are exact, so the result is that of the whole)
__device__ __forceinline__ float normalised(float x, float2 st)
{
    return fmaf(x, .5f, -.5f * st.x) * (st.y + st.y);
}

template <int VEC>
__device__ __forceinline__ void add_values(const float *v, float first, double &s, double &q)
{
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const double d = (double)v[i] - (double)first;
        s += d;
        q = fma(d, d, q);
    }
}

// The values of a chunk: into the checkpoint and into y.
template <int TYPE, bool KEEP>
__device__ __forceinline__ void put_values(const Fwd &a, typename Elem<TYPE>::T *y, int r, int col,
                                           v4u c, float2 st, const float *sc, const float *b)
{
    constexpr int VEC = Row<TYPE>::VEC;
    const int left = a.features - col;
    float n[VEC];
    chunk_values<TYPE>(c, n);
#pragma unroll
    for (int i = 0; i < VEC; ++i) n[i] = normalised(n[i], st);
    if (KEEP) {
        if (left < VEC) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) n[i] = i < left ? n[i] : 0.f;
        }
        keep_values<VEC>(a.k, (size_t)r * a.k.width + col, n);
    }
    if (!y) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i) n[i] = n[i] * sc[i] + b[i];
    write_values<TYPE>(y + r * a.y_stride + col, left, n, a.past);
}

template <int TYPE, int G, int I, bool KEEP>
__global__ void __launch_bounds__(G < 256 ? 256 : G)
k_norm_fwd(const typename Elem<TYPE>::T *x, typename Elem<TYPE>::T *y, Fwd a)
{
    constexpr int VEC = Row<TYPE>::VEC, NT = G < 256 ? 256 : G, AT_ONCE = NT / G;
    // (registers: 1024 threads have 128 each; with a checkpoint of 16-bit rows an address of
    // two lies in memory and is read back for each row)
    constexpr bool HOLD = I <= 2, AHEAD = G < 1024 || !KEEP;
    using T = typename Elem<TYPE>::T;
    __shared__ double sh[2][2 * NT / 64];
    const int t = threadIdx.x % G, step = (int)gridDim.x * AT_ONCE;
    int r = (int)blockIdx.x * AT_ONCE + threadIdx.x / G;
    float sc[HOLD ? I * VEC : VEC], b[HOLD ? I * VEC : VEC];
    auto parameters = [&](int c, float *s, float *o) {
        load_floats<VEC>(a.scales, c * VEC, a.features - c * VEC, 1.f, s);
        load_floats<VEC>(a.biases, c * VEC, a.features - c * VEC, 0.f, o);
    };
    if (HOLD && y) {
#pragma unroll
        for (int i = 0; i < I; ++i) parameters(t + i * G, sc + i * VEC, b + i * VEC);
    }
    v4u c[I], ahead[AHEAD ? I : 1];
    float first, next_first;
    auto load = [&](int row, v4u *to, float &f) {
        const T *p = x + row * a.stride;
        f = (float)p[0];
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int col = (t + i * G) * VEC;
            to[i] = load_chunk<TYPE>(p + col, a.features - col, f);
        }
    };
    if (r < a.rows) load(r, c, first);
    for (int turn = 0; r < a.rows; r += step, turn ^= 1) {
        const bool more = r + step < a.rows;
        if (AHEAD && more) load(r + step, ahead, next_first);
        double sums[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < I; ++i) {
            float v[VEC];
            chunk_values<TYPE>(c[i], v);
            add_values<VEC>(v, first, sums[0], sums[1]);
        }
        row_sums<G, 2>(sums, sh[turn]);
        if (I > 2) {
#pragma unroll
            for (int i = 0; i < I; ++i) forget(c[i]);
        }
        const float2 st = statistics(sums[0], sums[1], first, a.inv, a.eps);
        if (a.stats && t == 0) {
            a.stats[2 * (size_t)r] = st.x;
            a.stats[2 * (size_t)r + 1] = st.y;
        }
        if (y || KEEP) {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int at = t + i * G;
                if (at >= a.chunks) continue;
                if (!HOLD && y) parameters(at, sc, b);
                put_values<TYPE, KEEP>(a, y, r, at * VEC, c[i], st, sc + (HOLD ? i * VEC : 0),
                                       b + (HOLD ? i * VEC : 0));
            }
        }
        if (AHEAD) {
#pragma unroll
            for (int i = 0; i < I; ++i) c[i] = ahead[AHEAD ? i : 0];
            first = next_first;
        } else if (more) {
            load(r + step, c, first);
        }
    }
}

// Rows in parts: the sums of each part, then, from all of a row's, its values.
// A thread has FWD_U chunks (backward: BWD_U of delta and x) in flight, as the
// stores of one hold back the loads of the next (128 x 186624 fp32 forward 57 us with
// one, 53 with two, 51 with four; backward 128 and 92; 300 x 32768 bf16 backward 28 with
// two, 30 with four).
constexpr int PART_NT = 256, FWD_U = 4, BWD_U = 2;
constexpr int MOST_SPAN = 256;             // rows whose gradients' sums are one chain of additions
constexpr int MOST_GROUPS = (1 << 24) - 1;  // workgroups of a launch: for more values than a card holds
template <int TYPE>
__global__ void __launch_bounds__(PART_NT) k_norm_fwd_sums(const typename Elem<TYPE>::T *x, Fwd a)
{
    constexpr int VEC = Row<TYPE>::VEC;
    __shared__ double sh[2 * PART_NT / 64];
    const int r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const typename Elem<TYPE>::T *p = x + r * a.stride;
    const float first = (float)p[0];
    const int end = min((part + 1) * a.span, a.chunks);
    double sums[2] = {0, 0};
    for (int c = part * a.span + threadIdx.x; c < end; c += FWD_U * PART_NT) {
        v4u w[FWD_U];
#pragma unroll
        for (int u = 0; u < FWD_U; ++u) {
            const int at = min(c + u * PART_NT, end) * VEC;  // (behind the part: nothing but fill)
            w[u] = load_chunk<TYPE>(p + at, c + u * PART_NT < end ? a.features - at : 0, first);
        }
#pragma unroll
        for (int u = 0; u < FWD_U; ++u) {
            float v[VEC];
            chunk_values<TYPE>(w[u], v);
            add_values<VEC>(v, first, sums[0], sums[1]);
        }
    }
    row_sums<PART_NT, 2>(sums, sh);
    if (threadIdx.x == 0) {
        a.part[blockIdx.x] = make_double2(sums[0], sums[1]);
        if (part == 0) a.first[r] = first;  // (y may be x)
    }
}

template <int TYPE, bool KEEP>
__global__ void __launch_bounds__(PART_NT)
k_norm_fwd_values(const typename Elem<TYPE>::T *x, typename Elem<TYPE>::T *y, Fwd a)
{
    constexpr int VEC = Row<TYPE>::VEC;
    __shared__ double sh[2 * PART_NT / 64];
    const int r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const typename Elem<TYPE>::T *p = x + r * a.stride;
    const float first = a.first[r];
    double sums[2] = {0, 0};
    for (int i = threadIdx.x; i < a.parts; i += PART_NT) {
        const double2 v = a.part[(size_t)r * a.parts + i];
        sums[0] += v.x, sums[1] += v.y;
    }
    row_sums<PART_NT, 2>(sums, sh);
    const float2 st = statistics(sums[0], sums[1], first, a.inv, a.eps);
    if (a.stats && part == 0 && threadIdx.x == 0) {
        a.stats[2 * (size_t)r] = st.x;
        a.stats[2 * (size_t)r + 1] = st.y;
    }
    if (!y && !KEEP) return;
    const int end = min((part + 1) * a.span, a.chunks);
    for (int c = part * a.span + threadIdx.x; c < end; c += FWD_U * PART_NT) {
        v4u w[FWD_U];
        float sc[FWD_U][VEC], b[FWD_U][VEC];
#pragma unroll
        for (int u = 0; u < FWD_U; ++u) {
            const int col = (c + u * PART_NT) * VEC, left = c + u * PART_NT < end ? a.features - col : 0;
            w[u] = load_chunk<TYPE>(p + col, left, 0.f);
            if (y) {
                load_floats<VEC>(a.scales, col, left, 1.f, sc[u]);
                load_floats<VEC>(a.biases, col, left, 0.f, b[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < FWD_U; ++u) {
            const int at = c + u * PART_NT;
            if (at < end) put_values<TYPE, KEEP>(a, y, r, at * VEC, w[u], st, sc[u], b[u]);
        }
    }
}

// ---- backward -------------------------------------------------------------------------
struct Bwd {
    bool past;  // dx past the caches
    int rows, features, chunks;
    int64_t stride, d_stride, dx_stride;
    const float *stats, *scales;
    Kept k;
    float2 *sums;     // of rows in parts: [rows][parts] sums of g and of g*x_norm
    int parts, span;  // chunks of a part
    float *partial;   // [2][spans][features]: sums over rows, or null
    int rows_of, spans;  // rows of one (rows in parts), their number
    float *updates[2];   // of a single span, whose sums go there themselves; either may be null
    bool updating, accumulate;
};

// Where a span's sums over rows go: `which` 0 the scales', 1 the biases'.
__device__ __forceinline__ float *sums_of(const Bwd &a, int which, int span)
{
    if (!a.partial) return which ? a.updates[1] : a.updates[0];
    return a.partial + ((size_t)which * a.spans + span) * a.features;
}
template <int VEC>
__device__ __forceinline__ void store_sums(const Bwd &a, float *to, int left, float *v)
{
    if (a.accumulate) {
        float old[VEC];
        load_floats<VEC>(to, 0, left, 0.f, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += old[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; i += 4) store_values<ACH_F32>(to + i, left - i, v + i);
}

// What the sums and the values need of a row's chunk: delta and x as they lie in
// memory (or x_norm's codes and step).
template <int TYPE, bool KEPT> struct Pair {
    static constexpr int VEC = Row<TYPE>::VEC;
    using T = typename Elem<TYPE>::T;
    v4u d;
    uint32_t x[KEPT ? VEC / 4 : 4], step;
    __device__ __forceinline__ void load(const T *delta, const T *xs, const Bwd &a, int r, int col)
    {
        const int left = a.features - col;
        d = load_chunk<TYPE>(delta + r * a.d_stride + col, left, 0.f);
        if (KEPT) {
            // (codes behind the last value are 0, up to a whole block)
            const size_t at = (size_t)r * a.k.width + min(col, a.k.width - VEC);
            __builtin_memcpy(x, __builtin_assume_aligned(a.k.codes + at, VEC), VEC);
            step = a.k.steps[at / KEPT_BLOCK];
        } else {
            // (behind the last value delta is 0 and x one of the row's values: any
            // other's x_norm might be too large for a float)
            float fill = 0.f;
            if (left < VEC) fill = (float)xs[r * a.stride];
            const v4u c = load_chunk<TYPE>(xs + r * a.stride + col, left, fill);
            __builtin_memcpy(x, &c, sizeof(c));
        }
    }
    __device__ __forceinline__ void values(float2 st, float *dv, float *n) const
    {
        chunk_values<TYPE>(d, dv);
        if constexpr (KEPT) {
            const float scale = kept_scale(step);
#pragma unroll
            for (int i = 0; i < VEC; ++i) n[i] = (float)(int8_t)(x[i / 4] >> (8 * (i % 4))) * scale;
        } else {
            v4u c;
            __builtin_memcpy(&c, x, sizeof(c));
            chunk_values<TYPE>(c, n);
#pragma unroll
            for (int i = 0; i < VEC; ++i) n[i] = normalised(n[i], st);
        }
    }
};

__device__ __forceinline__ float2 stats_of(const Bwd &a, int r)
{
    return make_float2(a.stats[2 * (size_t)r], a.stats[2 * (size_t)r + 1]);
}

// A workgroup of 1024 threads has 128 registers each: with four chunks a thread and
// four ahead, the sums of the parameters' gradients lie in LDS (and, from a checkpoint, one
// value for after the rows in memory).
template <int G, int I> constexpr int bwd_lds()
{
    return G == 1024 && I == 4 ? 2 * 1024 * I * (int)sizeof(float4) : 0;
}

template <int TYPE, int G, int I, bool KEPT>
__global__ void __launch_bounds__(G < 256 ? 256 : G)
k_norm_bwd(const typename Elem<TYPE>::T *delta, const typename Elem<TYPE>::T *x,
           typename Elem<TYPE>::T *dx, Bwd a, float inv)
{
    constexpr int VEC = Row<TYPE>::VEC, NT = G < 256 ? 256 : G, AT_ONCE = NT / G;
    constexpr bool HOLD = G < 1024;  // (registers)
    constexpr bool IN_LDS = bwd_lds<G, I>() > 0;  // the gradients' sums: a float4 of each thread after the other
    using P = Pair<TYPE, KEPT>;
    __shared__ float sh[2][2 * NT / 64];
    __shared__ float join[AT_ONCE > 1 ? NT * I * VEC : 1];
    const int t = threadIdx.x % G, step = (int)gridDim.x * AT_ONCE;
    int r = (int)blockIdx.x * AT_ONCE + threadIdx.x / G;
    extern __shared__ __align__(16) float4 in_lds[];
    float sc[HOLD ? I * VEC : VEC], ds[IN_LDS ? VEC : I * VEC], db[IN_LDS ? VEC : I * VEC];
    if (HOLD) {
#pragma unroll
        for (int i = 0; i < I; ++i)
            load_floats<VEC>(a.scales, (t + i * G) * VEC, a.features - (t + i * G) * VEC, 1.f, sc + i * VEC);
    }
    if (IN_LDS) {
#pragma unroll
        for (int i = 0; i < 2 * I; ++i) in_lds[i * G + t] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
#pragma unroll
        for (int i = 0; i < I * VEC; ++i) ds[i] = db[i] = 0.f;
    }
    // a chunk's share of these sums, in turn with those of the row
    auto fetch = [&](int i) {
        if (!IN_LDS) return;
        __builtin_memcpy(ds, &in_lds[i * G + t], 16);
        __builtin_memcpy(db, &in_lds[(I + i) * G + t], 16);
    };
    auto put = [&](int i) {
        if (!IN_LDS) return;
        __builtin_memcpy(&in_lds[i * G + t], ds, 16);
        __builtin_memcpy(&in_lds[(I + i) * G + t], db, 16);
    };
    P c[I], ahead[I];
    float2 st, next;
    auto load = [&](int row, P *to, float2 &s) {
        s = stats_of(a, row);
#pragma unroll
        for (int i = 0; i < I; ++i) to[i].load(delta, x, a, row, (t + i * G) * VEC);
    };
    if (r < a.rows) load(r, c, st);
    for (int turn = 0; r < a.rows; r += step, turn ^= 1) {
        if (r + step < a.rows) load(r + step, ahead, next);
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < I; ++i) {
            float d[VEC], n[VEC];
            c[i].values(st, d, n);
            if (!HOLD && dx) load_floats<VEC>(a.scales, (t + i * G) * VEC, a.features - (t + i * G) * VEC, 1.f, sc);
            const int at = IN_LDS ? 0 : i * VEC;
            fetch(i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = d[e] * sc[(HOLD ? i * VEC : 0) + e];
                sums[0] += g;
                sums[1] = fmaf(g, n[e], sums[1]);
                ds[at + e] = fmaf(d[e], n[e], ds[at + e]);
                db[at + e] += d[e];
            }
            put(i);
        }
        if (dx) {
            row_sums<G, 2>(sums, sh[turn]);
            const float m1 = sums[0] * inv, m2 = sums[1] * inv;
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int col = (t + i * G) * VEC;
                if (col >= a.features) continue;
                float d[VEC], n[VEC];
                c[i].values(st, d, n);
                if (!HOLD) load_floats<VEC>(a.scales, col, a.features - col, 1.f, sc);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    d[e] = st.y * (d[e] * sc[(HOLD ? i * VEC : 0) + e] - m1 - n[e] * m2);
                write_values<TYPE>(dx + r * a.dx_stride + col, a.features - col, d, a.past);
            }
        }
#pragma unroll
        for (int i = 0; i < I; ++i) c[i] = ahead[i];
        st = next;
    }
    if (!a.updating) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float *const v = which ? db : ds;
        float *const to = sums_of(a, which, blockIdx.x);
        if (!to) continue;
        if (AT_ONCE > 1) {  // the workgroup's rows, in LDS as [value][row][thread]
            if (which) __syncthreads();
#pragma unroll
            for (int i = 0; i < I * VEC; ++i) join[i * NT + threadIdx.x] = v[i];
            __syncthreads();
            for (int j = threadIdx.x; j < G * I * VEC; j += NT) {
                const int i = j / G, u = j % G;
                const int col = (u + i / VEC * G) * VEC + i % VEC;
                if (col >= a.features) continue;
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) s += join[i * NT + k * G + u];
                to[col] = a.accumulate ? to[col] + s : s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int col = (t + i * G) * VEC;
                if (IN_LDS) __builtin_memcpy(v, &in_lds[(which * I + i) * G + t], 16);
                store_sums<VEC>(a, to + col, a.features - col, v + (IN_LDS ? 0 : i * VEC));
            }
        }
    }
}

// Rows in parts: the sums of each part, then tiles of columns over spans of rows.
template <int TYPE, bool KEPT>
__global__ void __launch_bounds__(PART_NT)
k_norm_bwd_sums(const typename Elem<TYPE>::T *delta, const typename Elem<TYPE>::T *x, Bwd a)
{
    constexpr int VEC = Row<TYPE>::VEC;
    __shared__ float sh[2 * PART_NT / 64];
    const int r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const float2 st = stats_of(a, r);
    const int end = min((part + 1) * a.span, a.chunks);
    float sums[2] = {0.f, 0.f};
    for (int c = part * a.span + threadIdx.x; c < end; c += BWD_U * PART_NT) {
        Pair<TYPE, KEPT> p[BWD_U];
        float sc[BWD_U][VEC];
#pragma unroll
        for (int u = 0; u < BWD_U; ++u) {
            // (behind the part: nothing of delta, so that it adds nothing)
            const bool in = c + u * PART_NT < end;
            const int col = (in ? c + u * PART_NT : a.chunks) * VEC;
            p[u].load(delta, x, a, r, col);
            load_floats<VEC>(a.scales, col, a.features - col, 1.f, sc[u]);
        }
#pragma unroll
        for (int u = 0; u < BWD_U; ++u) {
            float d[VEC], n[VEC];
            p[u].values(st, d, n);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = d[e] * sc[u][e];
                sums[0] += g;
                sums[1] = fmaf(g, n[e], sums[1]);
            }
        }
    }
    row_sums<PART_NT, 2>(sums, sh);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = make_float2(sums[0], sums[1]);
}

template <int TYPE, bool KEPT>
__global__ void __launch_bounds__(PART_NT)
k_norm_bwd_values(const typename Elem<TYPE>::T *delta, const typename Elem<TYPE>::T *x,
                  typename Elem<TYPE>::T *dx, Bwd a, float inv)
{
    constexpr int VEC = Row<TYPE>::VEC;
    const int tiles = (a.chunks + PART_NT - 1) / PART_NT;
    const int tile = blockIdx.x % tiles, span = blockIdx.x / tiles;
    const int col = (tile * PART_NT + threadIdx.x) * VEC, left = a.features - col;
    const int r0 = span * a.rows_of, end = min((int64_t)a.rows, (int64_t)r0 + a.rows_of);
    __shared__ float2 means[MOST_SPAN];  // of g and of g*x_norm
    if (dx) {
        const int lane = threadIdx.x & 63;
        for (int r = r0 + (threadIdx.x >> 6); r < end; r += PART_NT / 64) {
            double s1 = 0, s2 = 0;
            for (int i = lane; i < a.parts; i += 64) {
                const float2 v = a.sums[(size_t)r * a.parts + i];
                s1 += v.x, s2 += v.y;
            }
            s1 = wave_total(s1), s2 = wave_total(s2);
            if (lane == 63) means[r - r0] = make_float2((float)s1 * inv, (float)s2 * inv);
        }
        __syncthreads();
    }
    if (left <= 0) return;
    float sc[VEC], ds[VEC], db[VEC];
    load_floats<VEC>(a.scales, col, left, 1.f, sc);
#pragma unroll
    for (int e = 0; e < VEC; ++e) ds[e] = db[e] = 0.f;
    for (int r = r0; r < end; r += BWD_U) {
        Pair<TYPE, KEPT> p[BWD_U];
        float2 st[BWD_U];
#pragma unroll
        for (int u = 0; u < BWD_U; ++u)
            if (r + u < end) {
                st[u] = stats_of(a, r + u);
                p[u].load(delta, x, a, r + u, col);
            }
#pragma unroll
        for (int u = 0; u < BWD_U; ++u) {
            if (r + u >= end) break;
            float d[VEC], n[VEC];
            p[u].values(st[u], d, n);
#pragma unroll
            for (int e = 0; e < VEC; ++e) ds[e] = fmaf(d[e], n[e], ds[e]), db[e] += d[e];
            if (!dx) continue;
            const float2 m = means[r + u - r0];
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = st[u].y * (d[e] * sc[e] - m.x - n[e] * m.y);
            write_values<TYPE>(dx + (r + u) * a.dx_stride + col, left, d, a.past);
        }
    }
    if (!a.updating) return;
    float *const to = sums_of(a, 0, span), *const to_b = sums_of(a, 1, span);
    if (to) store_sums<VEC>(a, to + col, left, ds);
    if (to_b) store_sums<VEC>(a, to_b + col, left, db);
}

// The partial sums of a column: few by one thread, more by a thread in each of 16 waves.
template <int SHARES>
__global__ void __launch_bounds__(SHARES == 1 ? 256 : SHARES * 64)
k_norm_bwd_join(const float *partial, int spans, int features, float *scale_updates,
                float *bias_updates, int accumulate)
{
    constexpr int U = 8, COLS = SHARES == 1 ? 256 : 64;  // loads in flight, columns of a workgroup
    __shared__ double sh[SHARES][SHARES == 1 ? 1 : COLS];
    float *const to = blockIdx.y ? bias_updates : scale_updates;
    if (!to) return;
    const int lane = threadIdx.x % COLS, share = threadIdx.x / COLS;
    for (int first = blockIdx.x * COLS; first < features; first += (int)gridDim.x * COLS) {
        const int j = first + lane;
        double s = 0;
        if (j < features) {
            const float *p = partial + (size_t)blockIdx.y * spans * features + j;
            int i = share;
            for (; i + (U - 1) * SHARES < spans; i += U * SHARES) {
                float v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = p[(size_t)(i + u * SHARES) * features];
#pragma unroll
                for (int u = 0; u < U; ++u) s += v[u];
            }
            for (; i < spans; i += SHARES) s += p[(size_t)i * features];
        }
        if (SHARES > 1) {
            sh[share][lane] = s;
            __syncthreads();
            for (int n = SHARES / 2; n; n >>= 1) {
                if (share < n) sh[share][lane] = s += sh[share + n][lane];
                __syncthreads();
            }
        }
        if (share == 0 && j < features) to[j] = accumulate ? (float)(to[j] + s) : (float)s;
    }
}

// ---- plans ---------------------------------------------------------------------------
bool layernorm_desc(const ach_layernorm_desc *d, ach_layernorm_desc *out)
{
    if (!d || d->rows < 0 || d->features < 1 || d->features > KEPT_MOST || d->stride < 0) return false;
    if (d->rows > KEPT_MOST || !elem_type(d->type) || !(d->eps >= 1e-12f && d->eps <= 1.f)) return false;
    *out = *d;
    if (out->stride == 0) out->stride = d->features;
    return out->stride >= d->features;
}

bool row_stride(int64_t *stride, int features)
{
    if (*stride == 0) *stride = features;
    return *stride >= features;
}

int tiles_of(int n, int tile) { return (n + tile - 1) / tile; }
size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

bool past_caches(const ach_layernorm_desc &d)
{
    return (size_t)d.rows * d.features * elem_size(d.type) > (size_t)16 << 20;
}

// Chunks of a row, in whole blocks of a checkpoint.
int chunks_of(const ach_layernorm_desc &d)
{
    const int vec = 16 / (int)elem_size(d.type);
    return (int)(((int64_t)d.features + KEPT_BLOCK - 1) / KEPT_BLOCK * KEPT_BLOCK / vec);
}

struct Plan {
    int grid;            // workgroups of rows in registers; 0: rows in parts
    int parts, span;     // of a row: parts, chunks of each
    int tiles, rows_of, spans;  // backward, rows in parts: tiles of columns, rows of a span, spans
    size_t first, partial, bytes;  // of the workspace
};

// The threads that share a row and the chunks of each: the fewest threads that
// hold it.
template <int G_, int I_> struct Kind {
    static constexpr int G = G_, I = I_, NT = G < 256 ? 256 : G;
};
template <class F> bool for_kind(int chunks, int most, F f)
{
    if (chunks > most) return false;
    if (chunks <= 16) f(Kind<16, 1>());
    else if (chunks <= 64) f(Kind<64, 1>());
    else if (chunks <= 128) f(Kind<64, 2>());
    else if (chunks <= 256) f(Kind<256, 1>());
    else if (chunks <= 512) f(Kind<256, 2>());
    else if (chunks <= 1024) f(Kind<512, 2>());
    else if (chunks <= 2048) f(Kind<512, 4>());
    else f(Kind<1024, 4>());
    return true;
}
template <class F> bool for_bwd_kind(int chunks, int most, F f)
{
    if (chunks > most) return false;
    if (chunks <= 16) f(Kind<16, 1>());
    else if (chunks <= 64) f(Kind<64, 1>());
    else if (chunks <= 128) f(Kind<64, 2>());
    else if (chunks <= 256) f(Kind<256, 1>());
    else if (chunks <= 512) f(Kind<256, 2>());
    else if (chunks <= 1024) f(Kind<512, 2>());
    else if (chunks <= 1536) f(Kind<768, 2>());
    else if (chunks <= 2048) f(Kind<1024, 2>());
    else f(Kind<1024, 4>());
    return true;
}
// A row's chunks that fit the registers, four of each thread's, which a workgroup
// of 1024 has 128 of; the backward pass holds two sums for each value, those of 8
// values a chunk for two chunks.  (Twice as many in the forward pass, eight
// chunks a thread: 1000 x 60000 bf16 91 us, in parts 73.)
constexpr int FWD_CHUNKS = 4096;
constexpr int bwd_chunks(int type) { return type == ACH_F32 ? 4096 : 2048; }

void in_parts(int chunks, int rows, Plan *p)
{
    // parts of 2 to 16 chunks a thread, so that there are 1024 workgroups where that can be
    int64_t parts = rows ? 1024 / rows : 1;
    const int64_t least = (chunks + 16 * PART_NT - 1) / (16 * PART_NT), most = chunks / (2 * PART_NT);
    if (parts > most) parts = most;
    if (parts < least) parts = least;
    if (parts < 1) parts = 1;
    p->span = (int)((chunks + parts - 1) / parts);
    p->span = (p->span + PART_NT - 1) / PART_NT * PART_NT;
    p->parts = (chunks + p->span - 1) / p->span;
}

Plan fwd_plan(const ach_layernorm_desc &d)
{
    Plan p = {};
    const int chunks = chunks_of(d);
    if (!for_kind(chunks, FWD_CHUNKS, [&](auto k) {
            const int at_once = k.NT / k.G, all = (d.rows + at_once - 1) / at_once;
            // (512 or 1024 threads: two a compute unit, whose parameters serve several rows;
            // 1000 x 16000 bf16 16 us, with 1024 workgroups 18, with 256 20)
            p.grid = min(all, k.NT >= 512 ? 512 : 2048);
        })) {
        in_parts(chunks, d.rows, &p);
        p.first = (size_t)d.rows * p.parts * sizeof(double2);
        p.bytes = p.first + (size_t)d.rows * sizeof(float);
    }
    return p;
}

Plan bwd_plan(const ach_layernorm_desc &d)
{
    Plan p = {};
    const int chunks = chunks_of(d);
    if (!for_bwd_kind(chunks, bwd_chunks(d.type), [&](auto k) {
            const int at_once = k.NT / k.G, all = (d.rows + at_once - 1) / at_once;
            // Two a compute unit.  One of those whose registers fill it (1024 and 768 threads, 512
            // with 16-bit rows: 300 x 8000 fp16 14 us, two 17, four chunks of each of 256 threads
            // 18), and one of 512 threads with fp32 rows, which would share it, where the partial
            // sums are a large part of the work (700 x 3000 12 and 13, 10000 rows 91 and 71).
            // More, where a chain of sums would be longer than 256 rows.
            const bool one = k.NT > 512 || (k.NT == 512 && (d.type != ACH_F32 || d.rows <= 1024));
            p.grid = min(all, max(one ? 256 : 512, (all + 255) / 256));
            // of 1024 threads no more than take equally many turns (1027 x 13001 with 206
            // instead of 256, 43 -> 40 us; 700 x 3000 fp32 with 234 12 -> 13)
            if (k.NT == 1024 && p.grid) p.grid = tiles_of(all, tiles_of(all, p.grid));
            // a second launch costs more than a second turn (2 x 4096 fp32 7.4 us, in two
            // workgroups 9.9), but for the largest (2 x 16000 fp32 10.5 and 9.7)
            if (k.NT < 1024 && all == 2) p.grid = 1;
            p.spans = p.grid;
        })) {
        in_parts(chunks, d.rows, &p);
        p.tiles = (chunks + PART_NT - 1) / PART_NT;
        const int spans = d.rows <= 4 ? 1 : min(max(1024 / p.tiles, tiles_of(d.rows, MOST_SPAN)), d.rows);
        p.rows_of = d.rows ? (int)(((int64_t)d.rows + spans - 1) / spans) : 1;
        p.spans = (int)(((int64_t)d.rows + p.rows_of - 1) / p.rows_of);
        p.partial = round16((size_t)d.rows * p.parts * sizeof(float2));
    }
    p.bytes = p.partial + (size_t)2 * p.spans * d.features * sizeof(float);  // (a single span's: unused)
    return p;
}

template <int TYPE, bool KEEP>
int fwd_go(const Plan &p, const void *x, void *y, const Fwd &a, int chunks, hipStream_t st)
{
    using T = typename Elem<TYPE>::T;
    if (!for_kind(chunks, FWD_CHUNKS, [&](auto k) {
            hipLaunchKernelGGL((k_norm_fwd<TYPE, k.G, k.I, KEEP>), dim3(p.grid), dim3(k.NT), 0, st,
                               (const T *)x, (T *)y, a);
        })) {
        const dim3 grid((unsigned)(a.rows * p.parts)), nt(PART_NT);
        hipLaunchKernelGGL((k_norm_fwd_sums<TYPE>), grid, nt, 0, st, (const T *)x, a);
        hipLaunchKernelGGL((k_norm_fwd_values<TYPE, KEEP>), grid, nt, 0, st, (const T *)x, (T *)y, a);
    }
    return check_launch();
}

template <int TYPE, bool KEPT>
int bwd_go(const Plan &p, const void *delta, const void *x, void *dx, const Bwd &a, int chunks,
           hipStream_t st)
{
    using T = typename Elem<TYPE>::T;
    const float inv = (float)(1. / a.features);
    int rc = ACH_OK;
    if (!for_bwd_kind(chunks, bwd_chunks(TYPE), [&](auto k) {
            if constexpr (k.G * k.I <= bwd_chunks(TYPE)) {
                constexpr int lds = bwd_lds<k.G, k.I>();
                const auto kern = &k_norm_bwd<TYPE, k.G, k.I, KEPT>;
                if (lds > 64 * 1024)
                    rc = check(hipFuncSetAttribute(reinterpret_cast<const void *>(kern),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, lds));
                if (rc) return;
                hipLaunchKernelGGL(kern, dim3(p.grid), dim3(k.NT), lds, st, (const T *)delta,
                                   (const T *)x, (T *)dx, a, inv);
            }
        })) {
        if (dx)
            hipLaunchKernelGGL((k_norm_bwd_sums<TYPE, KEPT>), dim3((unsigned)(a.rows * p.parts)),
                               dim3(PART_NT), 0, st, (const T *)delta, (const T *)x, a);
        hipLaunchKernelGGL((k_norm_bwd_values<TYPE, KEPT>), dim3((unsigned)(p.tiles * p.spans)),
                           dim3(PART_NT), 0, st, (const T *)delta, (const T *)x, (T *)dx, a, inv);
    }
    return rc ? rc : check_launch();
}

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_layernorm_fwd_workspace(const ach_layernorm_desc *desc)
{
    ach_layernorm_desc d;
    return layernorm_desc(desc, &d) ? fwd_plan(d).bytes : 0;
}

int ach_layernorm_fwd(const ach_layernorm_desc *desc, const void *x, const float *scales,
                      const float *biases, void *y, int64_t y_stride, float *stats,
                      void *checkpoint, void *ws, size_t ws_bytes, ach_stream_t s)
{
    ach_layernorm_desc d;
    if (!layernorm_desc(desc, &d) || !x || (!y && !stats && !checkpoint)) return ACH_EINVAL;
    if (!row_stride(&y_stride, d.features)) return ACH_EINVAL;
    const size_t size = elem_size(d.type);
    if (!aligned(x, size) || !aligned(y, size) || !aligned(checkpoint, 16)) return ACH_EINVAL;
    if (!aligned(scales, 4) || !aligned(biases, 4) || !aligned(stats, 4)) return ACH_EINVAL;
    if (y == x && y_stride != d.stride) return ACH_EINVAL;
    const Plan p = fwd_plan(d);
    if (p.bytes && (!ws || ws_bytes < p.bytes || !aligned(ws, 16))) return ACH_EWORKSPACE;
    if (d.rows == 0) return ACH_OK;
    Fwd a = {past_caches(d), d.rows, d.features, 0, 1. / d.features, d.eps, d.stride, y_stride, scales, biases,
             stats, {}, (double2 *)ws, (float *)((char *)ws + p.first), p.parts, p.span};
    if (checkpoint) a.k = kept(checkpoint, d.rows, d.features);
    hipStream_t st = as_stream(s);
    const int vec = 16 / (int)size;
    a.chunks = checkpoint ? chunks_of(d) : (d.features + vec - 1) / vec;
    if ((int64_t)d.rows * p.parts > MOST_GROUPS) return ACH_EINVAL;
#define CALL(TYPE)                                                                                 \
    return checkpoint ? fwd_go<TYPE, true>(p, x, y, a, chunks_of(d), st)                           \
                      : fwd_go<TYPE, false>(p, x, y, a, chunks_of(d), st)
    FOR_TYPE(d.type, CALL);
#undef CALL
}

size_t ach_layernorm_bwd_workspace(const ach_layernorm_desc *desc)
{
    ach_layernorm_desc d;
    return layernorm_desc(desc, &d) ? bwd_plan(d).bytes : 0;
}

int ach_layernorm_bwd(const ach_layernorm_desc *desc, const void *delta, int64_t delta_stride,
                      const void *x, const void *checkpoint, const float *stats,
                      const float *scales, void *dx, int64_t dx_stride, float *scale_updates,
                      float *bias_updates, int accumulate, void *ws, size_t ws_bytes,
                      ach_stream_t s)
{
    ach_layernorm_desc d;
    if (!layernorm_desc(desc, &d) || !delta || !stats || !x == !checkpoint) return ACH_EINVAL;
    if ((!dx && !scale_updates && !bias_updates) || (accumulate != 0 && accumulate != 1))
        return ACH_EINVAL;
    if (!row_stride(&delta_stride, d.features) || !row_stride(&dx_stride, d.features))
        return ACH_EINVAL;
    const size_t size = elem_size(d.type);
    if (!aligned(delta, size) || !aligned(x, size) || !aligned(dx, size)) return ACH_EINVAL;
    if (!aligned(checkpoint, 16) || !aligned(stats, 4) || !aligned(scales, 4)) return ACH_EINVAL;
    if (!aligned(scale_updates, 4) || !aligned(bias_updates, 4)) return ACH_EINVAL;
    if (dx == delta && dx_stride != delta_stride) return ACH_EINVAL;
    const Plan p = bwd_plan(d);
    const bool updating = scale_updates || bias_updates, joined = updating && p.spans != 1;
    const size_t bytes = updating ? p.bytes : p.partial;  // (without updates no sums over rows)
    if (bytes && (!ws || ws_bytes < bytes || !aligned(ws, 16))) return ACH_EWORKSPACE;
    if ((int64_t)d.rows * p.parts > MOST_GROUPS || (int64_t)p.tiles * p.spans > MOST_GROUPS)
        return ACH_EINVAL;
    hipStream_t st = as_stream(s);
    float *const partial = joined ? (float *)((char *)ws + p.partial) : nullptr;
    const int vec = 16 / (int)size;
    if (d.rows) {
        Bwd a = {past_caches(d), d.rows, d.features, (d.features + vec - 1) / vec, d.stride, delta_stride, dx_stride,
                 stats, scales, {}, (float2 *)ws, p.parts, p.span, partial, p.rows_of, p.spans,
                 {scale_updates, bias_updates}, updating, accumulate && !joined};
        if (checkpoint) a.k = kept(checkpoint, d.rows, d.features);
        int rc;
#define CALL(TYPE)                                                                                 \
    rc = checkpoint ? bwd_go<TYPE, true>(p, delta, x, dx, a, chunks_of(d), st)                     \
                    : bwd_go<TYPE, false>(p, delta, x, dx, a, chunks_of(d), st)
        FOR_TYPE(d.type, CALL);
#undef CALL
        if (rc) return rc;
    }
    if (joined) {
        // few of them are one thread's (4 x 1000000 fp32 by 16 waves each: 84 us in all, 26 so)
        const bool few = p.spans <= 32;
        const int tiles = tiles_of(d.features, few ? 256 : 64);
        hipLaunchKernelGGL(few ? &k_norm_bwd_join<1> : &k_norm_bwd_join<16>,
                           dim3((unsigned)min(tiles, 1 << 20), 2), dim3(few ? 256 : 1024), 0, st,
                           (const float *)partial, p.spans, d.features, scale_updates, bias_updates,
                           accumulate);
        return check_launch();
    }
    return ACH_OK;
}

}  // extern "C"
