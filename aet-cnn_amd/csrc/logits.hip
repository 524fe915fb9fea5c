// Operators on rows of logits (include/aetcnn_ops.h): log probabilities of
// given classes with entropy and top alternatives, their gradient, and
// distillation from a teacher's top logits.
#include "common.hpp"

#include <float.h>
#include <math.h>

namespace ach {
namespace {

template <int TYPE> struct Elem;
template <> struct Elem<ACH_F32> {
    using T = float;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
template <> struct Elem<ACH_BF16> {
    using T = __bf16;
    static __device__ __forceinline__ float get(T v) { return (float)v; }
    static __device__ __forceinline__ T put(float v) { return (T)v; }
};
template <> struct Elem<ACH_F16> {
    using T = _Float16;
    static __device__ __forceinline__ float get(T v) { return (float)v; }
    static __device__ __forceinline__ T put(float v) { return (T)v; }
};

// Order of logits: larger values have larger keys, -0 equals +0.
__device__ __forceinline__ uint32_t order_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ ((u & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}

// Combines v over the 256 threads; every thread gets the result.
template <class V, class F> __device__ V block_all(V v, V *sh, F f)
{
    for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return f(f(sh[0], sh[1]), f(sh[2], sh[3]));
}

template <int TYPE>
__global__ void __launch_bounds__(256)
    k_logprobs(ach_logits_desc d, const typename Elem<TYPE>::T *__restrict__ logits,
               const int32_t *__restrict__ ids, int k, float *logprobs, int32_t *ranks,
               float *entropy, float *stats, int32_t *top_ids, float *top_logprobs)
{
    __shared__ double shd[4];
    __shared__ float shf[4];
    __shared__ int shi[4];
    __shared__ unsigned long long shu[4];
    const auto addd = [](double a, double b) { return a + b; };
    const auto maxf = [](float a, float b) { return fmaxf(a, b); };
    const auto maxu = [](unsigned long long a, unsigned long long b) { return a > b ? a : b; };
    const int n = d.classes;
    const float inv_t = 1.f / d.temperature;
    for (int r = blockIdx.x; r < d.rows; r += gridDim.x) {
        const auto *row = logits + (size_t)r * d.stride;
        float m = -INFINITY;
        for (int j = threadIdx.x; j < n; j += 256) m = fmaxf(m, Elem<TYPE>::get(row[j]));
        m = block_all(m, shf, maxf);
        int first = n;  // the first class of logit m, which the sum leaves out: its exponential is 1
        for (int j = threadIdx.x; j < n && first == n; j += 256)
            if (Elem<TYPE>::get(row[j]) == m) first = j;
        first = block_all(first, shi, [](int a, int b) { return a < b ? a : b; });
        const int id = ids ? ids[r] : -1;
        const bool given = id >= 0 && id < n;
        const float x_id = given ? Elem<TYPE>::get(row[id]) : 0.f;
        const float ref = m == -INFINITY ? 0.f : m;
        double s = 0, t = 0, above = 0;
        for (int j = threadIdx.x; j < n; j += 256) {
            const float x = Elem<TYPE>::get(row[j]);
            const float z = (x - ref) * inv_t, e = expf(z);
            if (j != first) s += e;
            if (e != 0.f) t += (double)e * z;
            above += x > x_id;
        }
        s = block_all(s, shd, addd);
        t = block_all(t, shd, addd);
        above = block_all(above, shd, addd);
        const bool bad = !(s < INFINITY) || m == INFINITY;  // a NaN or a +inf in the row
        if (bad) s = NAN;
        const bool empty = m == -INFINITY && !bad;
        const float log_s = empty ? -INFINITY : (float)log1p(s);
        if (threadIdx.x == 0) {
            if (logprobs)
                logprobs[r] = !given ? 0.f : empty ? -INFINITY : (x_id - m) * inv_t - log_s;
            if (ranks) ranks[r] = !given || bad ? -1 : (int)above;
            if (entropy) entropy[r] = empty ? 0.f : (float)(log1p(s) - t / (1 + s));
            if (stats) {
                stats[2 * (size_t)r] = bad ? NAN : m;
                stats[2 * (size_t)r + 1] = log_s;
            }
        }
        unsigned long long last = ~0ull;
        for (int i = 0; i < k; ++i) {
            unsigned long long best = 0;
            for (int j = threadIdx.x; j < n; j += 256) {
                const unsigned long long c =
                    ((unsigned long long)order_key(Elem<TYPE>::get(row[j])) << 32) |
                    (uint32_t)~j;
                if (c < last && c > best) best = c;
            }
            last = block_all(best, shu, maxu);
            if (threadIdx.x == 0) {
                const int j = (int)~(uint32_t)last;
                const float x = Elem<TYPE>::get(row[bad ? 0 : j]);
                top_ids[(size_t)r * k + i] = bad ? -1 : j;
                top_logprobs[(size_t)r * k + i] =
                    bad ? NAN : empty ? -INFINITY : (x - m) * inv_t - log_s;
            }
        }
    }
}

template <int TYPE>
__global__ void __launch_bounds__(256)
    k_logprobs_bwd(ach_logits_desc d, const typename Elem<TYPE>::T *logits,
                   const int32_t *__restrict__ ids, const float *__restrict__ stats,
                   const float *__restrict__ entropy, const float *__restrict__ dlogprobs,
                   const float *__restrict__ dentropy, typename Elem<TYPE>::T *dlogits,
                   int64_t dstride)
{
    const int n = d.classes;
    const float inv_t = 1.f / d.temperature;
    for (int r = blockIdx.x; r < d.rows; r += gridDim.x) {
        const auto *row = logits + (size_t)r * d.stride;
        auto *out = dlogits + (size_t)r * dstride;
        const int id = ids ? ids[r] : -1;
        const float g = dlogprobs && id >= 0 && id < n ? dlogprobs[r] : 0.f;
        const float h = dentropy ? dentropy[r] : 0.f;
        const float m = stats[2 * (size_t)r], log_s = stats[2 * (size_t)r + 1];
        const float ent = dentropy ? entropy[r] : 0.f;
        const bool none = (g == 0.f && h == 0.f) || m == -INFINITY;
        for (int j = threadIdx.x; j < n; j += 256) {
            float v = 0.f;
            if (!none) {
                const float logp = (Elem<TYPE>::get(row[j]) - m) * inv_t - log_s;
                const float p = expf(logp);
                v = j == id ? -g * expm1f(logp) : -g * p;
                if (p != 0.f) v -= h * p * (logp + ent);
                v *= inv_t;
            }
            out[j] = Elem<TYPE>::put(v);
        }
    }
}

// The listed classes of a row in a distillation: the teacher's, and the label.
struct Listed {
    int id;      // -1: dropped
    int teacher; // whether the teacher lists it
    double p;    // the teacher's probability
    float x;     // the student's logit
};

__device__ float load_any(const void *p, int type, size_t i)
{
    return type == ACH_F32 ? ((const float *)p)[i]
           : type == ACH_BF16 ? (float)((const __bf16 *)p)[i]
                              : (float)((const _Float16 *)p)[i];
}

template <int TYPE>
__global__ void __launch_bounds__(256)
    k_distill(ach_logits_desc d, ach_distill_desc t, const typename Elem<TYPE>::T *logits,
              const int32_t *__restrict__ teacher_ids, const void *__restrict__ teacher_values,
              const int32_t *__restrict__ labels, const float *__restrict__ row_weights,
              float *loss, typename Elem<TYPE>::T *delta, int64_t delta_stride, float *row_loss)
{
    __shared__ Listed list[ACH_TOP_MAX + 1];
    __shared__ double shd[4];
    __shared__ float shf[4];
    const auto addd = [](double a, double b) { return a + b; };
    const auto maxf = [](float a, float b) { return fmaxf(a, b); };
    const int n = d.classes, k = t.soft != 0.f ? t.k : 0;
    const bool tail = t.mode == ACH_DISTILL_TAIL;
    const double inv_t = 1. / d.temperature;
    for (int r = blockIdx.x; r < d.rows; r += gridDim.x) {
        const auto *row = logits + (size_t)r * d.stride;
        const float w = row_weights ? row_weights[r] : 1.f;
        if (w == 0.f) {
            if (delta)
                for (int j = threadIdx.x; j < n; j += 256)
                    delta[(size_t)r * delta_stride + j] = Elem<TYPE>::put(0.f);
            if (threadIdx.x == 0) {
                if (loss) loss[r] = 0.f;
                if (row_loss) row_loss[r] = 0.f;
            }
            continue;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            double vmax = -INFINITY, sum = 0;
            for (int i = 0; i < k; ++i) {
                int id = teacher_ids[(size_t)r * k + i];
                if (id < 0 || id >= n) id = -1;
                for (int l = 0; l < i && id >= 0; ++l)
                    if (list[l].id == id) id = -1;
                double v = load_any(teacher_values, t.teacher_type, (size_t)r * k + i);
                if (!tail) v *= inv_t;
                list[i] = {id, id >= 0, id >= 0 ? v : 0, id >= 0 ? Elem<TYPE>::get(row[id]) : 0.f};
                if (id >= 0 && !(v <= vmax)) vmax = v;
            }
            for (int i = 0; i < k; ++i) {
                if (list[i].id < 0) continue;
                list[i].p = tail ? exp(list[i].p) : vmax == -INFINITY ? 0 : exp(list[i].p - vmax);
                sum += list[i].p;
            }
            if (!tail && sum != 0)
                for (int i = 0; i < k; ++i) list[i].p /= sum;
            int y = t.hard != 0.f && labels ? labels[r] : -1;
            if (y < 0 || y >= n) y = -1;
            list[k] = {y, 0, 0, y >= 0 ? Elem<TYPE>::get(row[y]) : 0.f};
        }
        __syncthreads();
        const int y = list[k].id;
        const float x_y = list[k].x;
        bool y_listed = false;
        float m = -INFINITY, mo = -INFINITY;  // of all classes, of those not listed
        for (int j = threadIdx.x; j < n; j += 256) {
            const float x = Elem<TYPE>::get(row[j]);
            bool listed = false;
            for (int i = 0; i <= k; ++i) listed |= list[i].id == j;
            m = fmaxf(m, x);
            if (!listed) mo = fmaxf(mo, x);
        }
        m = block_all(m, shf, maxf);
        mo = block_all(mo, shf, maxf);
        const float ref = m == -INFINITY ? 0.f : m, refo = mo == -INFINITY ? 0.f : mo;
        double so = 0, so1 = 0;
        for (int j = threadIdx.x; j < n; j += 256) {
            const float x = Elem<TYPE>::get(row[j]);
            bool listed = false;
            for (int i = 0; i <= k; ++i) listed |= list[i].id == j;
            if (listed) continue;
            so += exp((x - refo) * inv_t);
            so1 += exp((double)(x - refo));
        }
        so = block_all(so, shd, addd);
        so1 = block_all(so1, shd, addd);
        const double up = mo == -INFINITY ? 0 : exp(((double)refo - ref) * inv_t),
                     up1 = mo == -INFINITY ? 0 : exp((double)refo - ref);
        double total = so * up, total1 = so1 * up1, sp = 0, kd = 0, tail_sum = so * up;
        for (int i = 0; i < k; ++i) {
            if (list[i].id < 0) continue;
            if (list[i].id == y) y_listed = true;
            total += exp(((double)list[i].x - ref) * inv_t);
            total1 += exp((double)list[i].x - ref);
            sp += list[i].p;
        }
        if (y >= 0 && !y_listed) {
            total += exp(((double)x_y - ref) * inv_t);
            total1 += exp((double)x_y - ref);
            tail_sum += exp(((double)x_y - ref) * inv_t);
        }
        const bool empty = m == -INFINITY && total == 0;
        const double lse = log(total);
        for (int i = 0; i < k; ++i)
            if (list[i].id >= 0 && list[i].p != 0)
                kd += list[i].p * (log(list[i].p) - (((double)list[i].x - ref) * inv_t - lse));
        double P = sp, rest = 0, a_tail = 0;
        if (tail && k > 0 && tail_sum != 0) {
            rest = sp > 1 ? 0 : 1 - sp;
            if (rest != 0) kd += rest * (log(rest) - (log(tail_sum) - lse));
            P += rest;
            a_tail = rest / tail_sum;
        }
        double row_value = t.soft * (double)d.temperature * d.temperature * kd;
        if (k == 0) row_value = 0;
        if (y >= 0) row_value += t.hard * (log(total1) - ((double)x_y - ref));
        if (empty) row_value = 0;
        if (threadIdx.x == 0) {
            if (loss) loss[r] = (float)(w * row_value);
            if (row_loss) row_loss[r] = (float)(w * row_value);
        }
        if (!delta) continue;
        const double soft = k > 0 ? (double)t.soft * d.temperature : 0, hard = y >= 0 ? t.hard : 0;
        for (int j = threadIdx.x; j < n; j += 256) {
            const float x = Elem<TYPE>::get(row[j]);
            double p = 0;
            bool mine = false;
            for (int i = 0; i < k; ++i)
                if (list[i].id == j) {
                    mine = true;
                    p = list[i].p;
                }
            const double e = exp(((double)x - ref) * inv_t), e1 = exp((double)x - ref);
            double g = 0;
            if (soft != 0) g += soft * (P * e / total - p - (mine ? 0 : a_tail * e));
            if (hard != 0) g += hard * (e1 / total1 - (j == y));
            delta[(size_t)r * delta_stride + j] = Elem<TYPE>::put(empty ? 0.f : (float)(-w * g));
        }
    }
}

__global__ void __launch_bounds__(256) k_sum_losses(const float *__restrict__ row_loss, int rows,
                                                    float *cost)
{
    __shared__ double sh[4];
    double s = 0;
    for (int i = threadIdx.x; i < rows; i += 256) s += row_loss[i];
    s = block_all(s, sh, [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) *cost = (float)s;
}

size_t elem_size(int type) { return type == ACH_F32 ? 4 : 2; }

bool aligned(const void *p, size_t size) { return ((uintptr_t)p & (size - 1)) == 0; }

// The descriptor with its stride filled in; false if it describes nothing.
bool logits_desc(const ach_logits_desc *d, ach_logits_desc *out)
{
    if (!d || d->rows < 0 || d->classes <= 0 || d->stride < 0) return false;
    if (d->type != ACH_F32 && d->type != ACH_BF16 && d->type != ACH_F16) return false;
    if (!(d->temperature >= 1e-6f && d->temperature <= 1e6f)) return false;
    *out = *d;
    if (out->stride == 0) out->stride = d->classes;
    return out->stride >= d->classes;
}

bool distill_desc(const ach_distill_desc *t, int classes)
{
    if (!t || !(fabsf(t->soft) < INFINITY) || !(fabsf(t->hard) < INFINITY)) return false;
    if (t->k < 0 || t->k > ACH_TOP_MAX || (t->soft != 0.f && t->k == 0)) return false;
    if (t->mode != ACH_DISTILL_RENORM && t->mode != ACH_DISTILL_TAIL) return false;
    return t->teacher_type == ACH_F32 || t->teacher_type == ACH_BF16 || t->teacher_type == ACH_F16;
}

unsigned row_grid(int rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_logprobs_workspace(const ach_logits_desc *desc, int k)
{
    return 0;
}

int ach_logprobs_fwd(const ach_logits_desc *desc, const void *logits, const int32_t *ids, int k,
                     float *logprobs, int32_t *ranks, float *entropy, float *stats,
                     int32_t *top_ids, float *top_logprobs, void *ws, size_t ws_bytes,
                     ach_stream_t s)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || k < 0 || k > ACH_TOP_MAX || k > d.classes) return ACH_EINVAL;
    if (!logits || !aligned(logits, elem_size(d.type))) return ACH_EINVAL;
    if ((logprobs || ranks) && !ids) return ACH_EINVAL;
    if (k > 0 && (!top_ids || !top_logprobs)) return ACH_EINVAL;
    if (k == 0 && !logprobs && !ranks && !entropy && !stats) return ACH_EINVAL;
    if (d.rows == 0) return ACH_OK;
    const dim3 grid(row_grid(d.rows)), block(256);
    hipStream_t st = as_stream(s);
#define LAUNCH(TYPE)                                                                              \
    hipLaunchKernelGGL((k_logprobs<TYPE>), grid, block, 0, st, d,                                 \
                       (const Elem<TYPE>::T *)logits, ids, k, logprobs, ranks, entropy, stats,    \
                       top_ids, top_logprobs)
    if (d.type == ACH_F32) LAUNCH(ACH_F32);
    else if (d.type == ACH_BF16) LAUNCH(ACH_BF16);
    else LAUNCH(ACH_F16);
#undef LAUNCH
    return check_launch();
}

int ach_logprobs_bwd(const ach_logits_desc *desc, const void *logits, const int32_t *ids,
                     const float *stats, const float *entropy, const float *dlogprobs,
                     const float *dentropy, void *dlogits, int64_t dstride, ach_stream_t s)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || !logits || !stats || !dlogits) return ACH_EINVAL;
    if (!aligned(logits, elem_size(d.type)) || !aligned(dlogits, elem_size(d.type)))
        return ACH_EINVAL;
    if ((!dlogprobs && !dentropy) || (dlogprobs && !ids) || (dentropy && !entropy))
        return ACH_EINVAL;
    if (dstride == 0) dstride = d.classes;
    if (dstride < d.classes || (dlogits == logits && dstride != d.stride)) return ACH_EINVAL;
    if (d.rows == 0) return ACH_OK;
    const dim3 grid(row_grid(d.rows)), block(256);
    hipStream_t st = as_stream(s);
#define LAUNCH(TYPE)                                                                              \
    hipLaunchKernelGGL((k_logprobs_bwd<TYPE>), grid, block, 0, st, d,                             \
                       (const Elem<TYPE>::T *)logits, ids, stats, entropy, dlogprobs, dentropy,   \
                       (Elem<TYPE>::T *)dlogits, dstride)
    if (d.type == ACH_F32) LAUNCH(ACH_F32);
    else if (d.type == ACH_BF16) LAUNCH(ACH_BF16);
    else LAUNCH(ACH_F16);
#undef LAUNCH
    return check_launch();
}

size_t ach_distill_workspace(const ach_logits_desc *desc, const ach_distill_desc *t)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || !distill_desc(t, d.classes)) return 0;
    return (size_t)d.rows * sizeof(float);
}

int ach_distill_xent(const ach_logits_desc *desc, const ach_distill_desc *t, const void *logits,
                     const int32_t *teacher_ids, const void *teacher_values,
                     const int32_t *labels, const float *row_weights, float *loss, void *delta,
                     int64_t delta_stride, float *cost, void *ws, size_t ws_bytes,
                     ach_stream_t s)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || !distill_desc(t, d.classes)) return ACH_EINVAL;
    if (!logits || !aligned(logits, elem_size(d.type))) return ACH_EINVAL;
    if (!loss && !delta && !cost) return ACH_EINVAL;
    if (t->soft != 0.f && (!teacher_ids || !teacher_values)) return ACH_EINVAL;
    if (teacher_values && !aligned(teacher_values, elem_size(t->teacher_type))) return ACH_EINVAL;
    if (t->hard != 0.f && !labels) return ACH_EINVAL;
    if (!aligned(delta, elem_size(d.type))) return ACH_EINVAL;
    if (delta_stride == 0) delta_stride = d.classes;
    if (delta && (delta_stride < d.classes || (delta == logits && delta_stride != d.stride)))
        return ACH_EINVAL;
    if (d.rows > 0 && (!ws || ws_bytes < ach_distill_workspace(desc, t))) return ACH_EWORKSPACE;
    hipStream_t st = as_stream(s);
    if (d.rows > 0) {
        const dim3 grid(row_grid(d.rows)), block(256);
#define LAUNCH(TYPE)                                                                              \
    hipLaunchKernelGGL((k_distill<TYPE>), grid, block, 0, st, d, *t,                              \
                       (const Elem<TYPE>::T *)logits, teacher_ids, teacher_values, labels,        \
                       row_weights, loss, (Elem<TYPE>::T *)delta, delta_stride, (float *)ws)
        if (d.type == ACH_F32) LAUNCH(ACH_F32);
        else if (d.type == ACH_BF16) LAUNCH(ACH_BF16);
        else LAUNCH(ACH_F16);
#undef LAUNCH
        const int rc = check_launch();
        if (rc || !cost) return rc;
    }
    if (!cost) return ACH_OK;
    hipLaunchKernelGGL(k_sum_losses, dim3(1), dim3(256), 0, st, (const float *)ws, d.rows, cost);
    return check_launch();
}

}  // extern "C"
