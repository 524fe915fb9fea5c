// Layer norm (include/aetcnn_ops.h): forward, and backward with the reduction of
// the scales' and biases' gradients.
#include "checkpoint.hpp"

#include <math.h>

namespace ach {
namespace {

constexpr int NT = 256;

// Sum over the workgroup; every thread gets it.  sh holds a V per wave and may
// be used again at once.
template <class V> __device__ __forceinline__ V block_sum(V v, V *sh)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    V r = sh[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) r += sh[i];
    return r;
}

// The reciprocal standard deviation.  Squares that pass a float's range, of
// differences from 1.8e19 on, are summed in 64 bits instead: `again` does that.
template <class F> __device__ __forceinline__ float rstd_of(float squares, float n, float eps, F again)
{
    if (squares < INFINITY) return 1.f / sqrtf(squares / n + eps);
    return (float)(1. / sqrt(again() / n + (double)eps));
}

struct Fwd {
    int rows, features, chunks;  // chunks of a row: with a checkpoint, of whole blocks
    float eps;
    int64_t stride, y_stride;
    const float *scales, *biases;
    float *stats;
    Kept k;
};

// A workgroup per row: sums relative to the row's first value (which keeps a
// mean far above the deviations exact), squares about the mean, then the values.
template <int TYPE, bool KEEP>
__global__ void __launch_bounds__(NT)
k_norm_fwd(const typename Elem<TYPE>::T *x, typename Elem<TYPE>::T *y, Fwd a)
{
    constexpr int VEC = Row<TYPE>::VEC;
    __shared__ float sh[NT / 64];
    __shared__ double shd[NT / 64];
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const typename Elem<TYPE>::T *p = x + r * a.stride;
        const float first = (float)p[0];
        auto each = [&](auto f) {
            for (int c = threadIdx.x; c < a.chunks; c += NT) {
                float v[VEC];
                load_values<TYPE>(p + c * VEC, a.features - c * VEC, v);
                f(c * VEC, v);
            }
        };
        float s = 0.f;
        each([&](int col, const float *v) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += col + i < a.features ? v[i] - first : 0.f;
        });
        const float mean = first + block_sum(s, sh) / (float)a.features;
        float q = 0.f;
        each([&](int col, const float *v) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = col + i < a.features ? v[i] - mean : 0.f;
                q += d * d;
            }
        });
        const float rstd = rstd_of(block_sum(q, sh), (float)a.features, a.eps, [&] {
            double t = 0;
            each([&](int col, const float *v) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const double d = col + i < a.features ? v[i] - mean : 0.f;
                    t += d * d;
                }
            });
            return block_sum(t, shd);
        });
        if (a.stats && threadIdx.x == 0) a.stats[2 * (size_t)r] = mean, a.stats[2 * (size_t)r + 1] = rstd;
        if (!y && !KEEP) continue;
        __syncthreads();  // y may be x, whose first value the others may still read
        each([&](int col, const float *v) {
            float n[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) n[i] = col + i < a.features ? (v[i] - mean) * rstd : 0.f;
            if (KEEP) keep_values<VEC>(a.k, (size_t)r * a.k.width + col, n);
            if (!y) return;
            float sc[VEC], b[VEC];
            load_floats<VEC>(a.scales, col, a.features - col, 1.f, sc);
            load_floats<VEC>(a.biases, col, a.features - col, 0.f, b);
#pragma unroll
            for (int i = 0; i < VEC; ++i) n[i] = n[i] * sc[i] + b[i];
            store_values<TYPE>(y + r * a.y_stride + col, a.features - col, n);
        });
    }
}

struct Bwd {
    int rows, features, chunks;
    int64_t stride, d_stride, dx_stride;
    const float *stats, *scales;
    Kept k;
    float2 *sums;   // [rows] {sum g, sum g*x_norm} / n
    float *part;    // [2][spans][features]
    int span, spans;  // rows of a partial sum
};

// x_norm of a chunk, from the rows or from their checkpoint
template <int TYPE, bool KEPT>
__device__ __forceinline__ void normal_values(const typename Elem<TYPE>::T *x, const Bwd &a, int r,
                                              int col, float mean, float rstd, float *v)
{
    constexpr int VEC = Row<TYPE>::VEC;
    if (KEPT) {
        kept_values<VEC>(a.k, (size_t)r * a.k.width + col, v);
        return;
    }
    load_values<TYPE>(x + r * a.stride + col, a.features - col, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (v[i] - mean) * rstd;
}

template <int TYPE, bool KEPT>
__global__ void __launch_bounds__(NT)
k_norm_bwd_sums(const typename Elem<TYPE>::T *delta, const typename Elem<TYPE>::T *x, Bwd a)
{
    constexpr int VEC = Row<TYPE>::VEC;
    __shared__ float sh[NT / 64];
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float mean = a.stats[2 * (size_t)r], rstd = a.stats[2 * (size_t)r + 1];
        float s = 0.f, t = 0.f;
        for (int c = threadIdx.x; c < a.chunks; c += NT) {
            const int col = c * VEC, left = a.features - col;
            float d[VEC], n[VEC], sc[VEC];
            load_values<TYPE>(delta + r * a.d_stride + col, left, d);
            normal_values<TYPE, KEPT>(x, a, r, col, mean, rstd, n);
            load_floats<VEC>(a.scales, col, left, 1.f, sc);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float g = d[i] * sc[i];
                if (i < left) s += g, t += g * n[i];
            }
        }
        s = block_sum(s, sh), t = block_sum(t, sh);
        if (threadIdx.x == 0) a.sums[r] = make_float2(s / a.features, t / a.features);
    }
}

// A tile of NT chunks of columns and a span of rows
template <int TYPE, bool KEPT>
__global__ void __launch_bounds__(NT)
k_norm_bwd_apply(const typename Elem<TYPE>::T *delta, const typename Elem<TYPE>::T *x,
                 typename Elem<TYPE>::T *dx, Bwd a)
{
    constexpr int VEC = Row<TYPE>::VEC;
    const int tiles = (a.chunks + NT - 1) / NT;
    const int tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
    const int col = (tile * NT + threadIdx.x) * VEC, left = a.features - col;
    if (left <= 0) return;
    float sc[VEC], ds[VEC], db[VEC];
    load_floats<VEC>(a.scales, col, left, 1.f, sc);
#pragma unroll
    for (int i = 0; i < VEC; ++i) ds[i] = db[i] = 0.f;
    const int end = min((int64_t)a.rows, (int64_t)(part + 1) * a.span);
    for (int r = part * a.span; r < end; ++r) {
        const float mean = a.stats[2 * (size_t)r], rstd = a.stats[2 * (size_t)r + 1];
        float d[VEC], n[VEC];
        load_values<TYPE>(delta + r * a.d_stride + col, left, d);
        normal_values<TYPE, KEPT>(x, a, r, col, mean, rstd, n);
#pragma unroll
        for (int i = 0; i < VEC; ++i) ds[i] += d[i] * n[i], db[i] += d[i];
        if (!dx) continue;
        const float2 m = a.sums[r];
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[i] = rstd * (d[i] * sc[i] - m.x - n[i] * m.y);
        store_values<TYPE>(dx + r * a.dx_stride + col, left, d);
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        if (i < left) {
            a.part[(size_t)part * a.features + col + i] = ds[i];
            a.part[((size_t)a.spans + part) * a.features + col + i] = db[i];
        }
}

__global__ void __launch_bounds__(NT)
k_norm_bwd_join(const float *part, int spans, int features, float *scale_updates,
                float *bias_updates, int accumulate)
{
    const int j = blockIdx.x * NT + threadIdx.x;
    float *to = blockIdx.y ? bias_updates : scale_updates;
    if (j >= features || !to) return;
    double s = 0;
    for (int i = 0; i < spans; ++i) s += part[((size_t)blockIdx.y * spans + i) * features + j];
    to[j] = accumulate ? (float)(to[j] + s) : (float)s;
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

unsigned grid_of(size_t n) { return (unsigned)(n < (1u << 20) ? n : 1u << 20); }

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

struct Plan {
    int tiles, span, spans;
    size_t sums, bytes;  // of the workspace: the rows' sums, all
};

Plan bwd_plan(const ach_layernorm_desc &d)
{
    Plan p;
    const int vec = 16 / (int)elem_size(d.type);
    p.tiles = ((d.features + vec - 1) / vec + NT - 1) / NT;
    int spans = 1024 / p.tiles;
    if (spans < d.rows / 256) spans = d.rows / 256;  // short chains of sums
    if (spans > d.rows) spans = d.rows;
    if (spans < 1) spans = 1;
    p.span = d.rows ? (int)(((int64_t)d.rows + spans - 1) / spans) : 1;
    p.spans = (int)(((int64_t)d.rows + p.span - 1) / p.span);
    p.sums = round16((size_t)d.rows * sizeof(float2));
    p.bytes = p.sums + (size_t)2 * p.spans * d.features * sizeof(float);
    return p;
}

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_layernorm_fwd_workspace(const ach_layernorm_desc *)
{
    return 0;
}

int ach_layernorm_fwd(const ach_layernorm_desc *desc, const void *x, const float *scales,
                      const float *biases, void *y, int64_t y_stride, float *stats,
                      void *checkpoint, void *, size_t, ach_stream_t s)
{
    ach_layernorm_desc d;
    if (!layernorm_desc(desc, &d) || !x || (!y && !stats && !checkpoint)) return ACH_EINVAL;
    if (!row_stride(&y_stride, d.features)) return ACH_EINVAL;
    const size_t size = elem_size(d.type);
    if (!aligned(x, size) || !aligned(y, size) || !aligned(checkpoint, 16)) return ACH_EINVAL;
    if (!aligned(scales, 4) || !aligned(biases, 4) || !aligned(stats, 4)) return ACH_EINVAL;
    if (y == x && y_stride != d.stride) return ACH_EINVAL;
    if (d.rows == 0) return ACH_OK;
    Fwd a = {d.rows, d.features, 0, d.eps, d.stride, y_stride, scales, biases, stats, {}};
    if (checkpoint) a.k = kept(checkpoint, d.rows, d.features);
    hipStream_t st = as_stream(s);
#define CALL(TYPE)                                                                                 \
    do {                                                                                           \
        using T = Elem<TYPE>::T;                                                                   \
        constexpr int VEC = Row<TYPE>::VEC;                                                        \
        a.chunks = checkpoint ? a.k.width / VEC : (d.features + VEC - 1) / VEC;                    \
        if (checkpoint)                                                                            \
            hipLaunchKernelGGL((k_norm_fwd<TYPE, true>), dim3(grid_of(d.rows)), dim3(NT), 0, st,   \
                               (const T *)x, (T *)y, a);                                           \
        else                                                                                       \
            hipLaunchKernelGGL((k_norm_fwd<TYPE, false>), dim3(grid_of(d.rows)), dim3(NT), 0, st,  \
                               (const T *)x, (T *)y, a);                                           \
    } while (0)
    FOR_TYPE(d.type, CALL);
#undef CALL
    return check_launch();
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
    if (p.bytes && (!ws || ws_bytes < p.bytes || !aligned(ws, 16))) return ACH_EWORKSPACE;
    hipStream_t st = as_stream(s);
    const bool updates = scale_updates || bias_updates;
    if (d.rows) {
        Bwd a = {d.rows, d.features, 0, d.stride, delta_stride, dx_stride, stats, scales, {},
                 (float2 *)ws, updates ? (float *)((char *)ws + p.sums) : nullptr, p.span, p.spans};
        if (checkpoint) a.k = kept(checkpoint, d.rows, d.features);
#define GO(TYPE, KEPT)                                                                             \
    do {                                                                                           \
        using T = Elem<TYPE>::T;                                                                   \
        constexpr int VEC = Row<TYPE>::VEC;                                                        \
        a.chunks = (d.features + VEC - 1) / VEC;                                                   \
        if (dx)                                                                                    \
            hipLaunchKernelGGL((k_norm_bwd_sums<TYPE, KEPT>), dim3(grid_of(d.rows)), dim3(NT), 0,  \
                               st, (const T *)delta, (const T *)x, a);                             \
        hipLaunchKernelGGL((k_norm_bwd_apply<TYPE, KEPT>), dim3((unsigned)(p.tiles * p.spans)),    \
                           dim3(NT), 0, st, (const T *)delta, (const T *)x, (T *)dx, a);           \
    } while (0)
#define CALL(TYPE)                                                                                 \
    do {                                                                                           \
        if (checkpoint) GO(TYPE, true);                                                            \
        else GO(TYPE, false);                                                                      \
    } while (0)
        FOR_TYPE(d.type, CALL);
#undef CALL
#undef GO
        const int rc = check_launch();
        if (rc) return rc;
    }
    if (updates) {
        hipLaunchKernelGGL(k_norm_bwd_join, dim3((unsigned)((d.features + NT - 1) / NT), 2), dim3(NT),
                           0, st, (const float *)((char *)ws + p.sums), p.spans, d.features,
                           scale_updates, bias_updates, accumulate);
        return check_launch();
    }
    return ACH_OK;
}

}  // extern "C"
