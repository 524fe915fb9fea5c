// Operators on rows of logits (include/aetcnn_ops.h): log probabilities of
// given classes with entropy and top alternatives, their gradient, and
// distillation from a teacher's top logits.
//
// All three are bound by memory: a row is read once for its statistics (the
// running maximum and the sums of exponentials relative to it, rescaled when
// the maximum moves), and a gradient costs one more read, which the caches
// serve where rows are not too long, and one write.  A row belongs to one
// workgroup, or, where there are too few rows to fill the chip, to several
// whose partial results a second launch joins.
#include "common.hpp"

#include <float.h>
#include <math.h>

namespace ach {
namespace {

#ifndef UNROLL
#define UNROLL 4
#endif
#ifndef T64
#define T64 2048
#define T256 16384
#endif
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// An element type: 16 bytes of it as one load from any element's address.
template <int TYPE> struct Elem;
template <> struct Elem<ACH_F32> {
    using T = float;
};
template <> struct Elem<ACH_BF16> {
    using T = __bf16;
};
template <> struct Elem<ACH_F16> {
    using T = _Float16;
};
template <int TYPE> struct Row {
    using T = typename Elem<TYPE>::T;
    static constexpr int VEC = 16 / sizeof(T);
    typedef T Chunk __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
    static __device__ __forceinline__ Chunk load(const T *p) { return *(const Chunk *)p; }
    static __device__ __forceinline__ void store(T *p, Chunk v) { *(Chunk *)p = v; }
};

// Order of logits: larger values have larger keys, -0 equals +0.
__device__ __forceinline__ uint32_t order_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ ((u & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k)
{
    return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
// (logit, class) as one number: larger logits first, then lower classes.
__device__ __forceinline__ uint64_t compound(float x, int j)
{
    return ((uint64_t)order_key(x) << 32) | (uint32_t)~j;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Combines v over the wave; every lane gets the result.
template <class V, class F> __device__ __forceinline__ V wave_all(V v, F f)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    return v;
}

struct Add {
    template <class V> __device__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
    template <class V> __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};

// The same for 32 bits without the LDS crossbar: within rows of 16 lanes by
// shifts, then from row to row; lane 63 has seen all.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float old, float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL,
                                                      ROWS, 0xf, false));
}
__device__ __forceinline__ float lane_value(float v, int lane)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ float wave_total(float v)
{
    v += dpp<0x111, 0xf>(0.f, v);
    v += dpp<0x112, 0xf>(0.f, v);
    v += dpp<0x114, 0xf>(0.f, v);
    v += dpp<0x118, 0xf>(0.f, v);
    v += dpp<0x142, 0xa>(0.f, v);
    v += dpp<0x143, 0xc>(0.f, v);
    return lane_value(v, 63);
}
__device__ __forceinline__ float wave_most(float v)
{
    v = fmaxf(v, dpp<0x111, 0xf>(v, v));
    v = fmaxf(v, dpp<0x112, 0xf>(v, v));
    v = fmaxf(v, dpp<0x114, 0xf>(v, v));
    v = fmaxf(v, dpp<0x118, 0xf>(v, v));
    v = fmaxf(v, dpp<0x142, 0xa>(v, v));
    v = fmaxf(v, dpp<0x143, 0xc>(v, v));
    return lane_value(v, 63);
}

// Sum of v over the workgroup; every thread gets it.  sh holds one V per
// wave and may be used again at once.
template <int NT, class V> __device__ __forceinline__ V block_sum(V v, V *sh)
{
    v = wave_all(v, Add());
    if (NT == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    V r = sh[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) r += sh[i];
    return r;
}

// The part [begin, begin + len) of a row that a workgroup works on, as whole
// chunks, dealt to the threads in turn, and up to VEC - 1 single elements,
// one to each of the first threads.
template <int TYPE> struct Range {
    using T = typename Elem<TYPE>::T;
    const T *p;
    int begin, len;
    __device__ int chunks() const { return len / Row<TYPE>::VEC; }
    __device__ int rest() const { return len % Row<TYPE>::VEC; }
};

// ---- statistics ----------------------------------------------------------------
// A thread's running statistics of the logits it has seen: their maximum m
// (-FLT_MAX before the first finite one, which a logit of -inf leaves there:
// its exponential is 0 either way), s = sum exp2((x - m) c) and, for the
// entropy, t = sum exp2((x - m) c) (x - m) c; and its wave's count of logits
// above the given one.  A NaN or +inf makes s a NaN.
struct Stat {
    float m, s, t;
    int above;
};

// exponents below this give 0 in 32 bits; it keeps 0 * -inf out of t
constexpr float FAR = -200.f;

__device__ __forceinline__ void raise(Stat &a, float m, float c)
{
    const float d = fmaxf((a.m - m) * c, FAR), f = exp2_fast(d);
    a.t = f * (a.t + a.s * d);
    a.s *= f;
    a.m = m;
}

// N logits of each lane, all lanes taking part.  Masked logits make the plain
// sum for t a NaN, 0 * -inf: then it is formed again without them.
template <bool ENTROPY, bool RANK, int N>
__device__ __forceinline__ void absorb(Stat &a, const float (&x)[N], float c, float x_id)
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > a.m) raise(a, m, c);
    float t = a.t;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = (x[i] - a.m) * c, e = exp2_fast(d);
        a.s += e;
        if (ENTROPY) t = fmaf(e, d, t);
        if (RANK) a.above += __popcll(__ballot(x[i] > x_id));
    }
    if (ENTROPY) {
        if (t != t) {
            t = a.t;
            for (int i = 0; i < N; ++i) {
                const float d = fmaxf((x[i] - a.m) * c, FAR);
                t = fmaf(exp2_fast(d), d, t);
            }
        }
        a.t = t;
    }
}

template <int TYPE, int NT, bool ENTROPY, bool RANK>
__device__ __forceinline__ Stat stream(const Range<TYPE> &g, float c, float x_id)
{
    constexpr int V = Row<TYPE>::VEC, U = UNROLL;
    typedef typename Row<TYPE>::Chunk Chunk;
    Stat a = {-FLT_MAX, 0.f, 0.f, 0};
    const int n = g.chunks(), lane = threadIdx.x & 63;
    int q = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63);  // the wave's first chunk
    for (; q + (U - 1) * NT + 64 <= n; q += U * NT) {
        Chunk v[U];
        float x[U * V];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = Row<TYPE>::load(g.p + (size_t)(q + u * NT + lane) * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) x[u * V + i] = (float)v[u][i];
        absorb<ENTROPY, RANK>(a, x, c, x_id);
    }
    for (; q < n; q += NT) {
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = -INFINITY;
        if (q + lane < n) {
            const Chunk v = Row<TYPE>::load(g.p + (size_t)(q + lane) * V);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = (float)v[i];
        }
        absorb<ENTROPY, RANK>(a, x, c, x_id);
    }
    if (threadIdx.x < 64) {
        const float x[1] = {lane < g.rest() ? (float)g.p[(size_t)n * V + lane] : -INFINITY};
        absorb<ENTROPY, RANK>(a, x, c, x_id);
    }
    return a;
}

// The statistics of a range: m its maximum, rest = sum exp2((x - m) c)
// without one logit of value m, so that the log of the sum, log1p(rest),
// keeps its precision where one class has nearly all the probability.
struct Total {
    float m, rest, t;
    int above;
};

// A wave's statistics; `own` is the part of the sum of the first thread that
// has seen the maximum, whose exponential, 1, it contains.
struct WaveStat {
    float m, own, others, t;
    int above, owner;
};

template <int NT> struct StatLds {
    WaveStat wave[NT / 64];
    float rest;
};

// m is -inf where every logit is; rest is NaN where one is NaN or +inf.
template <int TYPE, int NT>
__device__ __forceinline__ Total total_of(const Range<TYPE> &g, Stat a, float c, StatLds<NT> &sh)
{
    constexpr int W = NT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    WaveStat w;
    w.m = wave_most(a.m);
    const int first = __ffsll((unsigned long long)__ballot(a.m == w.m)) - 1;
    raise(a, w.m, c);
    w.own = lane_value(a.s, first);
    w.others = wave_total(lane == first ? 0.f : a.s);
    w.t = wave_total(a.t);
    w.above = a.above;
    w.owner = wave * 64 + first;
    int owner_wave = 0;
    float m = w.m, others = w.others, own = w.own;
    Total r = {m, 0.f, w.t, w.above};
    if (W > 1) {
        if (lane == 0) sh.wave[wave] = w;
        __syncthreads();
        m = sh.wave[0].m;
#pragma unroll
        for (int i = 1; i < W; ++i)
            if (sh.wave[i].m > m) {
                m = sh.wave[i].m;
                owner_wave = i;
            }
        others = r.t = 0.f;
        r.above = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const WaveStat &v = sh.wave[i];
            const float d = fmaxf((v.m - m) * c, FAR), f = exp2_fast(d), s = v.own + v.others;
            others += i == owner_wave ? v.others : f * s;
            r.t += f * (v.t + s * d);
            r.above += v.above;
        }
        own = sh.wave[owner_wave].own;
        w.owner = sh.wave[owner_wave].owner;
    }
    r.m = m;
    r.rest = others + (own - 1.f);
    if (others + own == 0.f) {
        r.m = -INFINITY;
        r.rest = 0.f;
    } else if (others + own < 1.5f) {
        // own - 1 has lost what the owner's other logits add to its 1: the
        // owner's wave sums them again without it
        constexpr int V = Row<TYPE>::VEC;
        if (wave == owner_wave) {
            const int n = g.chunks(), rounds = w.owner < n ? (n - w.owner + NT - 1) / NT : 0;
            float s = 0.f, at_max = 0.f;
            for (int i = lane; i < rounds * V + 1; i += 64) {
                size_t j = (size_t)(w.owner + i / V * NT) * V + i % V;
                if (i == rounds * V) {  // its single element behind the chunks, if it has one
                    if (w.owner >= g.rest()) continue;
                    j = (size_t)n * V + w.owner;
                }
                const float x = (float)g.p[j];
                if (x == m) at_max += 1.f;
                else s += exp2_fast((x - m) * c);
            }
            r.rest = others + (wave_total(s) + (wave_total(at_max) - 1.f));
            if (W > 1 && lane == 0) sh.rest = r.rest;
        }
        if (W > 1) {
            __syncthreads();
            r.rest = sh.rest;
        }
    }
    return r;
}

// ---- the k largest ---------------------------------------------------------------
// The threads' maxima bound the k-th largest logit from below: each wave's
// ceil(k / waves)-th largest maximum has k logits at or above the least of
// these.  Only the threads whose maximum reaches that bound have seen
// candidates, so only their chunks are read again (from the caches), by all
// threads together.  Of random logits some k log(waves) + k pass; they are put
// in order by counting for each how many are before it.
template <int NT> struct TopLds {
    // logits above the bound, and at it
    static constexpr int CAP = NT == 64 ? 256 : 1024, EQUAL = NT == 64 ? 128 : 512;
    uint64_t list[CAP + EQUAL];
    uint64_t equal[EQUAL];
    uint32_t bound[NT / 64];
    int hot[NT];
    int sum[NT / 64];
    int nhot, nlist, nequal;
};

// f(x, class) for every logit that the hot threads have seen.
template <int TYPE, int NT, class F>
__device__ __forceinline__ void each_hot(const Range<TYPE> &g, const TopLds<NT> &sh, F f)
{
    constexpr int V = Row<TYPE>::VEC;
    const int n = g.chunks(), hot = sh.nhot, rounds = (n + NT - 1) / NT;
    for (int i = threadIdx.x; i < hot * rounds; i += NT) {
        const int q = i / hot * NT + sh.hot[i % hot];
        if (q >= n) continue;
        const typename Row<TYPE>::Chunk v = Row<TYPE>::load(g.p + (size_t)q * V);
#pragma unroll
        for (int e = 0; e < V; ++e) f((float)v[e], g.begin + q * V + e);
    }
    if (threadIdx.x < g.rest())
        f((float)g.p[(size_t)n * V + threadIdx.x], g.begin + n * V + (int)threadIdx.x);
}

// Leaves in sh.list a superset of the k largest of the range (k <= its
// length, no NaN) and returns its size; `mine` is the thread's maximum.
template <int TYPE, int NT>
__device__ int candidates(const Range<TYPE> &g, float mine, int k, TopLds<NT> &sh)
{
    constexpr int CAP = TopLds<NT>::CAP, EQUAL = TopLds<NT>::EQUAL, W = NT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nth = (k + W - 1) / W;
    const uint32_t key = order_key(mine);
    uint32_t bound = 0;  // 16 bits of it: lower is as right
    for (int b = 31; b >= 16; --b) {
        const uint32_t up = bound | (1u << b);
        if (__popcll(__ballot(key >= up)) >= nth) bound = up;
    }
    __syncthreads();
    if (lane == 0) sh.bound[wave] = bound;
    if (threadIdx.x == 0) sh.nhot = sh.nlist = sh.nequal = 0;
    __syncthreads();
    for (int i = 0; i < W; ++i) bound = min(bound, sh.bound[i]);
    // up to -FLT_MAX, where a thread that has seen -inf alone starts: anything
    float low = bound <= order_key(-FLT_MAX) ? -INFINITY : key_value(bound);
    const bool is_hot = mine >= low;
    const uint64_t ballot = __ballot(is_hot);
    int at = 0;
    if (lane == 0) at = atomicAdd(&sh.nhot, __popcll(ballot));
    at = __shfl(at, 0, 64);
    if (is_hot) sh.hot[at + __popcll(ballot & ((1ull << lane) - 1))] = threadIdx.x;
    __syncthreads();
    for (int round = 0;; ++round) {
        each_hot<TYPE, NT>(g, sh, [&](float x, int j) {
            if (x > low) {
                const int i = atomicAdd(&sh.nlist, 1);
                if (i < CAP) sh.list[i] = compound(x, j);
            } else if (x == low && low != -INFINITY) {
                const int i = atomicAdd(&sh.nequal, 1);
                if (i < EQUAL) sh.equal[i] = compound(x, j);
            }
        });
        __syncthreads();
        if (sh.nlist <= CAP) break;
        // Too many: the k-th largest itself, bit by bit.  No logits are above
        // it that are not among the k, so the next round is the last.
        uint32_t kth = 0;
        for (int b = 31; b >= 0; --b) {
            const uint32_t up = kth | (1u << b);
            int count = 0;
            each_hot<TYPE, NT>(g, sh, [&](float x, int) { count += order_key(x) >= up; });
            if (block_sum<NT>(count, sh.sum) >= k) kth = up;
        }
        low = key_value(kth);
        __syncthreads();
        if (threadIdx.x == 0) sh.nlist = sh.nequal = 0;
        __syncthreads();
    }
    const int above = sh.nlist, need = k - above, equal = sh.nequal;
    if (need <= 0) return above;
    if (equal <= EQUAL && low != -INFINITY) {
        for (int i = threadIdx.x; i < equal; i += NT) sh.list[above + i] = sh.equal[i];
        __syncthreads();
        return above + equal;
    }
    // The first `need` of many equal logits, in the order of the classes.
    int found = 0;
    for (int base = 0; base < g.len && found < need; base += NT) {
        const int j = base + threadIdx.x;
        const bool is = j < g.len && (float)g.p[j] == low;
        const uint64_t mask = __ballot(is);
        __syncthreads();
        if (lane == 0) sh.sum[wave] = __popcll(mask);
        __syncthreads();
        int before = found;
        for (int i = 0; i < W; ++i) {
            if (i < wave) before += sh.sum[i];
            found += sh.sum[i];
        }
        before += __popcll(mask & ((1ull << lane) - 1));
        if (is && before < need) sh.list[above + before] = compound(low, g.begin + j);
    }
    __syncthreads();
    return k;
}

// emit(place, compound) for the k largest of list[0..n), largest first.
template <int NT, class F>
__device__ __forceinline__ void in_order(const uint64_t *list, int n, int k, F emit)
{
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t v = list[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += list[j] > v;
        if (place < k) emit(place, v);
    }
}

// ---- log probabilities -------------------------------------------------------------
struct LogprobsOut {
    float *logprobs;
    int32_t *ranks;
    float *entropy, *stats;
    int32_t *top_ids;
    float *top_logprobs;
};

// A row's outputs but its alternatives; returns the log of its sum.
__device__ float write_row(const LogprobsOut &o, int r, const Total &a, bool given, float x_id,
                           float inv_t, bool first_thread)
{
    const bool bad = !(a.rest < INFINITY), empty = a.m == -INFINITY && !bad;
    const float log_s = empty ? -INFINITY : log1pf(a.rest);
    if (first_thread) {
        if (o.logprobs)
            o.logprobs[r] = !given ? 0.f : empty ? -INFINITY : (x_id - a.m) * inv_t - log_s;
        if (o.ranks) o.ranks[r] = !given || bad ? -1 : a.above;
        if (o.entropy) o.entropy[r] = empty ? 0.f : log_s - a.t * LN2 / (1.f + a.rest);
        if (o.stats) {
            o.stats[2 * (size_t)r] = bad ? NAN : a.m;
            o.stats[2 * (size_t)r + 1] = log_s;
        }
    }
    return log_s;
}

__device__ __forceinline__ void write_top(const LogprobsOut &o, size_t at, uint64_t v, float m,
                                          float inv_t, float log_s)
{
    o.top_ids[at] = (int)~(uint32_t)v;
    o.top_logprobs[at] =
        m == -INFINITY ? -INFINITY : (key_value((uint32_t)(v >> 32)) - m) * inv_t - log_s;
}

// One workgroup per row, or per part of a row (parts > 1), `span` classes
// each; the parts' totals and their k largest go to `part` and `lists`.
template <int TYPE, int NT, bool ENTROPY, bool RANK>
__global__ void __launch_bounds__(NT)
    k_logprobs(ach_logits_desc d, const typename Elem<TYPE>::T *__restrict__ logits,
               const int32_t *__restrict__ ids, int k, LogprobsOut o, int parts, int span,
               Total *__restrict__ part, uint64_t *__restrict__ lists)
{
    __shared__ StatLds<NT> st;
    __shared__ TopLds<NT> top;
    const float inv_t = 1.f / d.temperature, c = inv_t * LOG2E;
    for (size_t w = blockIdx.x; w < (size_t)d.rows * parts; w += gridDim.x) {
        const int r = (int)(w / parts), at = (int)(w % parts) * span;
        const auto *row = logits + (size_t)r * d.stride;
        const Range<TYPE> g = {row + at, at, min(span, d.classes - at)};
        const int id = ids ? ids[r] : -1;
        const bool given = id >= 0 && id < d.classes;
        const float x_id = given ? (float)row[id] : INFINITY;
        const Stat mine = stream<TYPE, NT, ENTROPY, RANK>(g, c, x_id);
        const Total a = total_of<TYPE, NT>(g, mine, c, st);
        const bool bad = !(a.rest < INFINITY);
        if (parts > 1) {
            if (threadIdx.x == 0) part[w] = a;
        }
        const float log_s = parts > 1 ? 0.f
                                      : write_row(o, r, a, given, x_id, inv_t, threadIdx.x == 0);
        if (k > 0 && bad) {
            for (int i = threadIdx.x; i < k && parts == 1; i += NT) {
                o.top_ids[(size_t)r * k + i] = -1;
                o.top_logprobs[(size_t)r * k + i] = NAN;
            }
        } else if (k > 0) {
            const int mk = min(k, g.len), n = candidates<TYPE, NT>(g, mine.m, mk, top);
            if (parts > 1) {
                in_order<NT>(top.list, n, mk, [&](int i, uint64_t v) { lists[w * k + i] = v; });
                for (int i = mk + threadIdx.x; i < k; i += NT) lists[w * k + i] = 0;
            } else {
                in_order<NT>(top.list, n, k, [&](int i, uint64_t v) {
                    write_top(o, (size_t)r * k + i, v, a.m, inv_t, log_s);
                });
            }
        }
        __syncthreads();
    }
}

// Joins the parts of a row.  Of the parts' lists, for every m the m-th largest
// of their ceil(k/m)-th entries bounds the k-th largest of all from below;
// with m = 1, 2, 4, ... parts no more than k (2 + log2 parts) entries pass
// the best of these bounds, however the large logits are spread.
constexpr int MOST_PARTS = 64;

template <int TYPE, int NT>
__global__ void __launch_bounds__(NT)
    k_logprobs_join(ach_logits_desc d, const typename Elem<TYPE>::T *__restrict__ logits,
                    const int32_t *__restrict__ ids, int k, LogprobsOut o, int parts,
                    const Total *__restrict__ part, const uint64_t *__restrict__ lists)
{
    const float inv_t = 1.f / d.temperature, c = inv_t * LOG2E;
    __shared__ uint64_t list[ACH_TOP_MAX * 8];
    __shared__ uint64_t bounds[8];
    __shared__ int n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = blockIdx.x; r < d.rows; r += gridDim.x) {
        // every wave joins the totals by itself
        Total a = {-INFINITY, 0.f, 0.f, 0};
        if (lane < parts) a = part[(size_t)r * parts + lane];
        const bool bad = __any(!(a.rest < INFINITY));
        const float m = wave_all(a.m, Max());
        const uint64_t at_max = __ballot(a.m == m && lane < parts);
        const int owner = at_max ? __ffsll((unsigned long long)at_max) - 1 : 0;
        const float z = m == -INFINITY ? 0.f : fmaxf((a.m - m) * c, FAR);
        const float f = a.m == -INFINITY ? 0.f : exp2_fast(z), s = 1.f + a.rest;
        const float mine = a.m == -INFINITY ? 0.f : lane == owner ? a.rest : s * f;
        Total t;
        t.m = m;
        t.rest = bad ? NAN : wave_all(mine, Add());
        t.t = wave_all(a.m == -INFINITY ? 0.f : f * (a.t + s * z), Add());
        t.above = wave_all(a.above, Add());
        const int id = ids ? ids[r] : -1;
        const bool given = id >= 0 && id < d.classes;
        const float x_id = given ? (float)logits[(size_t)r * d.stride + id] : 0.f;
        const float log_s = write_row(o, r, t, given, x_id, inv_t, threadIdx.x == 0);
        if (k == 0) continue;
        if (bad) {
            for (int i = threadIdx.x; i < k; i += NT) {
                o.top_ids[(size_t)r * k + i] = -1;
                o.top_logprobs[(size_t)r * k + i] = NAN;
            }
            continue;
        }
        const uint64_t *from = lists + (size_t)r * parts * k;
        __syncthreads();
        if (threadIdx.x < 8) bounds[threadIdx.x] = 0;
        if (threadIdx.x == 0) n = 0;
        __syncthreads();
        for (int b = wave; b < 7 && (1 << b) <= parts; b += NT / 64) {
            const int nth = (k + (1 << b) - 1) >> b;
            const uint64_t v = lane < parts ? from[lane * k + nth - 1] : 0;
            int before = 0;
            for (int i = 0; i < parts; ++i) {
                const uint64_t other = __shfl(v, i, 64);
                before += other > v || (other == v && i < lane);
            }
            if (lane < parts && before == (1 << b) - 1) bounds[b] = v;
        }
        __syncthreads();
        uint64_t low = 1;  // 0 fills up short lists
        for (int b = 0; b < 7; ++b) low = max(low, bounds[b]);
        for (int i = threadIdx.x; i < parts * k; i += NT) {
            const uint64_t v = from[i];
            if (v < low) continue;
            const int to = atomicAdd(&n, 1);
            if (to < ACH_TOP_MAX * 8) list[to] = v;
        }
        __syncthreads();
        in_order<NT>(list, min(n, ACH_TOP_MAX * 8), k, [&](int i, uint64_t v) {
            write_top(o, (size_t)r * k + i, v, m, inv_t, log_s);
        });
        __syncthreads();
    }
}

// Each workgroup writes `span` chunks of a row.  With l = log p,
// dx = p (a + b l) for a = -(g + h H)/T, b = -h/T; of the given class
// g (1 - p) = -g expm1(l), which keeps its precision where p is near 1.
template <int TYPE>
__global__ void __launch_bounds__(256)
    k_logprobs_bwd(ach_logits_desc d, const typename Elem<TYPE>::T *logits,
                   const int32_t *__restrict__ ids, const float *__restrict__ stats,
                   const float *__restrict__ entropy, const float *__restrict__ dlogprobs,
                   const float *__restrict__ dentropy, typename Elem<TYPE>::T *dlogits,
                   int64_t dstride, int parts, int span)
{
    using T = typename Elem<TYPE>::T;
    constexpr int V = Row<TYPE>::VEC;
    typedef typename Row<TYPE>::Chunk Chunk;
    const int chunks = d.classes / V, rest = d.classes % V;
    const float inv_t = 1.f / d.temperature, c = inv_t * LOG2E;
    for (size_t w = blockIdx.x; w < (size_t)d.rows * parts; w += gridDim.x) {
        const int r = (int)(w / parts), first = (int)(w % parts) * span;
        const T *row = logits + (size_t)r * d.stride;
        T *out = dlogits + (size_t)r * dstride;
        const int id = ids ? ids[r] : -1;
        const float g = dlogprobs && id >= 0 && id < d.classes ? dlogprobs[r] : 0.f;
        const float h = dentropy ? dentropy[r] : 0.f, ent = dentropy ? entropy[r] : 0.f;
        const float m = stats[2 * (size_t)r], log_s = stats[2 * (size_t)r + 1];
        const bool none = (g == 0.f && h == 0.f) || m == -INFINITY;
        const float a = -inv_t * (g + h * ent), b = -inv_t * h * LN2, off = -log_s * LOG2E;
        const auto grad = [&](float x, int j) {
            const float l = fmaf(x - m, c, off), p = exp2_fast(l);
            float v = p * fmaf(b, fmaxf(l, FAR), a);
            if (j == id && g != 0.f) {
                const float logp = (x - m) * inv_t - log_s;
                v = -inv_t * g * expm1f(logp) + p * fmaf(b, fmaxf(l, FAR), -inv_t * h * ent);
            }
            return v;
        };
        const int last = min(first + span, chunks);
        for (int q = first + threadIdx.x; q < last; q += 256) {
            Chunk v = {};
            if (!none) {
                const Chunk x = Row<TYPE>::load(row + (size_t)q * V);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = (T)grad((float)x[i], q * V + i);
            }
            Row<TYPE>::store(out + (size_t)q * V, v);
        }
        if (last == chunks && threadIdx.x < rest) {
            const int j = chunks * V + threadIdx.x;
            out[j] = none ? (T)0.f : (T)grad((float)row[j], j);
        }
    }
}

// ---- distillation ------------------------------------------------------------------
// A row's listed classes, the teacher's entries and the label, are few: their
// terms are computed in 64 bits.  All others enter through their maximum and
// their sums of exponentials alone, so the sum over what the teacher leaves
// out is a sum of these, not a difference of nearly equal sums.  With
// e_j = exp((x_j - mo)/T) relative to the maximum mo of the classes that are
// not listed, the delta of such a class is K e_j + K1 e1_j (e1: at
// temperature 1), and that of a listed one is written over it afterwards.
struct Entry {
    double p;  // the teacher's probability
    int id;    // -1: dropped
    float x;   // the student's logit
};

struct Dense {
    float m, s, s1;
};

template <bool TWO>
__device__ __forceinline__ void raise_dense(Dense &a, float m, float c)
{
    a.s *= exp2_fast(fmaxf((a.m - m) * c, FAR));
    if (TWO) a.s1 *= exp2_fast(fmaxf((a.m - m) * LOG2E, FAR));
    a.m = m;
}

template <bool TWO, int N>
__device__ __forceinline__ void absorb_dense(Dense &a, const float (&x)[N], float c)
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > a.m) raise_dense<TWO>(a, m, c);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        a.s += exp2_fast((x[i] - a.m) * c);
        if (TWO) a.s1 += exp2_fast((x[i] - a.m) * LOG2E);
    }
}

template <int NT> struct DistillLds {
    static constexpr int SEG = NT * 128;  // classes of one bitmap of listed classes
    uint32_t bits[SEG / 32];
    Entry entry[ACH_TOP_MAX];
    int dropped[ACH_TOP_MAX];
    Dense wave[NT / 64];
    // the row's constants, from one wave
    double ref, total, total1, P, mt, tail;
    float K, K1, loss;
    int y_listed;
};

template <int TYPE, int NT, bool TWO>
__device__ Dense stream_dense(const Range<TYPE> &all, float c, int k, int y, DistillLds<NT> &sh)
{
    constexpr int V = Row<TYPE>::VEC, U = UNROLL, SEG = DistillLds<NT>::SEG;
    Dense a = {-FLT_MAX, 0.f, 0.f};
    for (int at = 0; at < all.len; at += SEG) {
        const Range<TYPE> g = {all.p + at, all.begin + at, min(SEG, all.len - at)};
        __syncthreads();
        for (int i = threadIdx.x; i < (g.len + 31) / 32; i += NT) sh.bits[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i <= k; i += NT) {
            const int j = (i < k ? sh.entry[i].id : y) - g.begin;
            if (j >= 0 && j < g.len) atomicOr(&sh.bits[j >> 5], 1u << (j & 31));
        }
        __syncthreads();
        const int n = g.chunks();
        // the listed classes of a chunk read as masked
        const auto fetch = [&](const typename Row<TYPE>::Chunk &v, int q, float *x) {
            const uint32_t mask = (sh.bits[q * V >> 5] >> (q * V & 31)) & ((1u << V) - 1);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = (float)v[i];
            if (mask)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (mask >> i & 1) x[i] = -INFINITY;
        };
        int q = threadIdx.x;
        for (; q + (U - 1) * NT < n; q += U * NT) {
            typename Row<TYPE>::Chunk v[U];
            float x[U * V];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = Row<TYPE>::load(g.p + (size_t)(q + u * NT) * V);
#pragma unroll
            for (int u = 0; u < U; ++u) fetch(v[u], q + u * NT, x + u * V);
            absorb_dense<TWO>(a, x, c);
        }
        for (; q < n; q += NT) {
            float x[V];
            fetch(Row<TYPE>::load(g.p + (size_t)q * V), q, x);
            absorb_dense<TWO>(a, x, c);
        }
        if (threadIdx.x < g.rest()) {
            const int j = n * V + threadIdx.x;
            const bool listed = sh.bits[j >> 5] >> (j & 31) & 1;
            const float x[1] = {listed ? -INFINITY : (float)g.p[j]};
            absorb_dense<TWO>(a, x, c);
        }
    }
    raise_dense<TWO>(a, wave_most(a.m), c);
    a.s = wave_total(a.s);
    if (TWO) a.s1 = wave_total(a.s1);
    if (NT == 64) return a;
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = a;
    __syncthreads();
    a = sh.wave[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) {
        Dense b = sh.wave[i];
        const float m = fmaxf(a.m, b.m);
        raise_dense<TWO>(a, m, c);
        raise_dense<TWO>(b, m, c);
        a.s += b.s;
        if (TWO) a.s1 += b.s1;
    }
    return a;
}

__device__ __forceinline__ double load_any(const void *p, int type, size_t i)
{
    return type == ACH_F32    ? ((const float *)p)[i]
           : type == ACH_BF16 ? (float)((const __bf16 *)p)[i]
                              : (float)((const _Float16 *)p)[i];
}

// The teacher's entries of a row into sh.entry.
template <int TYPE, int NT>
__device__ void read_teacher(const typename Elem<TYPE>::T *row, int classes,
                             const int32_t *teacher_ids, const void *values, int type, size_t at,
                             int k, bool tail, double inv_t, DistillLds<NT> &sh)
{
    __syncthreads();
    for (int i = threadIdx.x; i < k; i += NT) {
        const int id = teacher_ids[at + i];
        const bool some = id >= 0 && id < classes;
        sh.entry[i].id = some ? id : -1;
        sh.entry[i].x = some ? (float)row[id] : 0.f;
        sh.dropped[i] = !some;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < k * k; i += NT) {  // repeated: the first one counts
        const int a = i / k, b = i % k;
        if (b < a && sh.entry[a].id == sh.entry[b].id) sh.dropped[a] = 1;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        double v[2], p[2], sum = 0, most = -INFINITY;
        for (int e = 0; e < 2; ++e) {
            const int i = threadIdx.x + e * 64;
            v[e] = i < k && !sh.dropped[i] ? load_any(values, type, at + i) : -INFINITY;
            if (!tail) v[e] *= inv_t;
            most = fmax(most, v[e]);
        }
        most = tail ? 0 : wave_all(most, Max());
        for (int e = 0; e < 2; ++e) {
            p[e] = v[e] == -INFINITY ? 0 : exp(v[e] - most);
            sum += p[e];
        }
        sum = wave_all(sum, Add());
        for (int e = 0; e < 2; ++e) {
            const int i = threadIdx.x + e * 64;
            if (i >= k) continue;
            sh.entry[i].p = tail || sum == 0 ? p[e] : p[e] / sum;
            if (sh.dropped[i]) sh.entry[i].id = -1;
        }
    }
    __syncthreads();
}

// The row's constants from its listed classes and the dense part, by the
// first wave.
template <int NT>
__device__ void constants(const Dense &a, const ach_distill_desc &t, int k, bool tail,
                          double temperature, int y, float x_y, float w, DistillLds<NT> &sh)
{
    if (threadIdx.x >= 64) return;
    const double inv_t = 1. / temperature;
    const int lane = threadIdx.x;
    float m = a.m;
    bool listed = false;
    for (int i = lane; i < k; i += 64)
        if (sh.entry[i].id >= 0) {
            m = fmaxf(m, sh.entry[i].x);
            listed |= sh.entry[i].id == y;
        }
    const bool y_listed = __any(listed);
    const bool extra = y >= 0 && !y_listed;  // the label as a class of its own
    m = wave_all(m, Max());
    if (y >= 0) m = fmaxf(m, x_y);
    const double ref = m;
    double total = 0, total1 = 0, sp = 0;
    for (int i = lane; i < k; i += 64)
        if (sh.entry[i].id >= 0) {
            const double z = sh.entry[i].x - ref;
            total += exp(z * inv_t);
            total1 += exp(z);
            sp += sh.entry[i].p;
        }
    total = wave_all(total, Add());
    total1 = wave_all(total1, Add());
    sp = wave_all(sp, Add());
    // without another class the dense part is empty: its sums are 0
    const double up = exp((a.m - ref) * inv_t), up1 = exp(a.m - ref);
    const double e_y = extra ? exp((x_y - ref) * inv_t) : 0;
    total += a.s * up + e_y;
    total1 += a.s1 * up1 + (extra ? exp(x_y - ref) : 0);
    const double lse = log(total);
    double kd = 0;
    for (int i = lane; i < k; i += 64) {
        const double p = sh.entry[i].p;
        if (sh.entry[i].id >= 0 && p != 0)
            kd += p * (log(p) - ((sh.entry[i].x - ref) * inv_t - lse));
    }
    kd = wave_all(kd, Add());
    // the rest: all classes that the teacher does not list, relative to their maximum mt
    const double mt = extra ? fmaxf(a.m, x_y) : a.m;
    const double sum_t = a.s * exp((a.m - mt) * inv_t) + (extra ? exp((x_y - mt) * inv_t) : 0);
    double P = sp, rest = 0;
    if (tail && k > 0 && sum_t != 0) {
        rest = sp > 1 ? 0 : 1 - sp;
        if (rest != 0) kd += rest * (log(rest) - (log(sum_t) + (mt - ref) * inv_t - lse));
        P += rest;
    }
    const double per_tail = rest == 0 ? 0 : rest / sum_t;
    double value = k > 0 ? t.soft * temperature * temperature * kd : 0;
    if (y >= 0) value += t.hard * (log(total1) - (x_y - ref));
    const bool empty = total == 0;
    const double soft = k > 0 ? -w * t.soft * temperature : 0, hard = y >= 0 ? -w * t.hard : 0;
    if (lane == 0) {
        sh.loss = empty ? 0.f : (float)(w * value);
        sh.K = empty || soft == 0 ? 0.f
                                  : (float)(soft * (P * up / total -
                                                    per_tail * exp((a.m - mt) * inv_t)));
        sh.K1 = empty || hard == 0 ? 0.f : (float)(hard * up1 / total1);
        sh.ref = ref;
        sh.total = empty ? INFINITY : total;
        sh.total1 = empty ? INFINITY : total1;
        sh.P = P;
        sh.mt = mt;
        sh.tail = per_tail;
        sh.y_listed = y_listed;
    }
}

// What a launch does: all of it, a row to a workgroup; or, for rows in parts,
// the statistics, then the delta.
enum { WHOLE, STATS, DELTA };

template <int TYPE, int NT, bool TWO, int MODE>
__global__ void __launch_bounds__(NT)
    k_distill(ach_logits_desc d, ach_distill_desc t, const typename Elem<TYPE>::T *logits,
              const int32_t *__restrict__ teacher_ids, const void *__restrict__ teacher_values,
              const int32_t *__restrict__ labels, const float *__restrict__ row_weights,
              float *loss, typename Elem<TYPE>::T *delta, int64_t delta_stride, float *row_loss,
              int parts, int span, Dense *dense, Entry *entries)
{
    using T = typename Elem<TYPE>::T;
    typedef typename Row<TYPE>::Chunk Chunk;
    constexpr int V = Row<TYPE>::VEC;
    __shared__ DistillLds<NT> sh;
    const int k = t.soft != 0.f ? t.k : 0;
    const bool tail = t.mode == ACH_DISTILL_TAIL;
    const float c = LOG2E / d.temperature;
    for (size_t b = blockIdx.x; b < (size_t)d.rows * parts; b += gridDim.x) {
        const int r = (int)(b / parts), part = (int)(b % parts), at = part * span;
        const T *row = logits + (size_t)r * d.stride;
        const Range<TYPE> g = {row + at, at, min(span, d.classes - at)};
        const float w = row_weights ? row_weights[r] : 1.f;
        if (MODE == STATS && w == 0.f) continue;
        int y = t.hard != 0.f ? labels[r] : -1;
        if (y >= d.classes) y = -1;
        if (w != 0.f) {
            Dense a;
            Entry *mine = MODE == WHOLE ? nullptr : entries + (size_t)r * (ACH_TOP_MAX + 1);
            float x_y = 0.f;
            if (MODE != DELTA) {
                x_y = y >= 0 ? (float)row[y] : 0.f;
                read_teacher<TYPE, NT>(row, d.classes, teacher_ids, teacher_values, t.teacher_type,
                                       (size_t)r * k, k, tail, 1. / d.temperature, sh);
                a = stream_dense<TYPE, NT, TWO>(g, c, k, y, sh);
                if (!TWO) a.s1 = a.s;
            }
            if (MODE == STATS) {
                if (threadIdx.x == 0) dense[b] = a;
                if (part == 0) {
                    for (int i = threadIdx.x; i < k; i += NT) mine[i] = sh.entry[i];
                    if (threadIdx.x == 0) mine[ACH_TOP_MAX].x = x_y;
                }
                __syncthreads();
                continue;
            }
            if (MODE == DELTA) {
                __syncthreads();
                for (int i = threadIdx.x; i < k; i += NT) sh.entry[i] = mine[i];
                x_y = y >= 0 ? mine[ACH_TOP_MAX].x : 0.f;
                const int lane = threadIdx.x & 63;
                a = {-FLT_MAX, 0.f, 0.f};
                if (lane < parts) a = dense[(size_t)r * parts + lane];
                const float m = wave_all(a.m, Max());
                raise_dense<true>(a, m, c);
                a.s = wave_all(a.s, Add());
                a.s1 = wave_all(a.s1, Add());
            }
            __syncthreads();
            constants<NT>(a, t, k, tail, d.temperature, y, x_y, w, sh);
            __syncthreads();
            if (threadIdx.x == 0 && part == 0) {
                if (loss) loss[r] = sh.loss;
                if (row_loss) row_loss[r] = sh.loss;
            }
            if (delta) {
                T *out = delta + (size_t)r * delta_stride + at;
                const float K = TWO ? sh.K : sh.K + sh.K1, K1 = sh.K1;
                const auto grad = [&](float x) {
                    float v = K * exp2_fast((x - a.m) * c);
                    if (TWO) v = fmaf(K1, exp2_fast((x - a.m) * LOG2E), v);
                    return v;
                };
                const int n = g.chunks();
                for (int q = threadIdx.x; q < n; q += NT) {
                    const Chunk x = Row<TYPE>::load(g.p + (size_t)q * V);
                    Chunk v;
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = (T)grad((float)x[i]);
                    Row<TYPE>::store(out + (size_t)q * V, v);
                }
                if (threadIdx.x < g.rest()) {
                    const int j = n * V + threadIdx.x;
                    out[j] = (T)grad((float)g.p[j]);
                }
                __syncthreads();  // the listed classes over what was written for them
                for (int i = threadIdx.x; i <= k; i += NT) {
                    const bool teacher = i < k;
                    const int id = teacher ? sh.entry[i].id : sh.y_listed ? -1 : y;
                    if (id < at || id >= at + g.len) continue;
                    const double x = teacher ? sh.entry[i].x : x_y, inv_t = 1. / d.temperature;
                    double v = 0;
                    if (k > 0) {
                        v = sh.P * exp((x - sh.ref) * inv_t) / sh.total;
                        v -= teacher ? sh.entry[i].p : sh.tail * exp((x - sh.mt) * inv_t);
                        v *= -w * t.soft * d.temperature;
                    }
                    if (y >= 0) v -= w * t.hard * (exp(x - sh.ref) / sh.total1 - (id == y));
                    if (sh.total == INFINITY) v = 0;  // no distribution
                    out[id - at] = (T)(float)v;
                }
            }
        } else {
            if (delta) {
                T *out = delta + (size_t)r * delta_stride + at;
                const Chunk zero = {};
                for (int q = threadIdx.x; q < g.chunks(); q += NT)
                    Row<TYPE>::store(out + (size_t)q * V, zero);
                if (threadIdx.x < g.rest()) out[g.chunks() * V + threadIdx.x] = (T)0.f;
            }
            if (threadIdx.x == 0 && part == 0) {
                if (loss) loss[r] = 0.f;
                if (row_loss) row_loss[r] = 0.f;
            }
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) k_sum_losses(const float *__restrict__ row_loss, int rows,
                                                    float *cost)
{
    __shared__ double sh[4];
    double s = 0;
    for (int i = threadIdx.x; i < rows; i += 256) s += row_loss[i];
    s = block_sum<256>(s, sh);
    if (threadIdx.x == 0) *cost = (float)s;
}

// ---- plans ---------------------------------------------------------------------------
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

bool distill_desc(const ach_distill_desc *t)
{
    if (!t || !(fabsf(t->soft) < INFINITY) || !(fabsf(t->hard) < INFINITY)) return false;
    if (t->k < 0 || t->k > ACH_TOP_MAX || (t->soft != 0.f && t->k == 0)) return false;
    if (t->mode != ACH_DISTILL_RENORM && t->mode != ACH_DISTILL_TAIL) return false;
    return t->teacher_type == ACH_F32 || t->teacher_type == ACH_BF16 || t->teacher_type == ACH_F16;
}

// Workgroups per row and the classes of each: one, unless the rows are few
// and long.
struct Split {
    int parts, span;
};

Split split_rows(int rows, int classes)
{
    int parts = rows > 0 ? 512 / rows : 1;
    parts = parts < classes / 4096 ? parts : classes / 4096;
    if (parts > MOST_PARTS) parts = MOST_PARTS;
    if (parts < 2) return {1, classes};
    const int span = (int)((((int64_t)classes + parts - 1) / parts + 63) / 64 * 64);
    return {(int)(((int64_t)classes + span - 1) / span), span};
}

// Threads of a workgroup for `span` classes; with k alternatives at least 2 k
// (the bound on the k-th largest is taken from the threads' maxima).
int threads_for(int span, int k)
{
    if (span <= T64 && k <= 32) return 64;
    return span <= T256 ? 256 : 1024;
}

unsigned grid_of(size_t n) { return (unsigned)(n < (1u << 20) ? n : 1u << 20); }

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace
}  // namespace ach

using namespace ach;

// CALL(TYPE) for the element type of a descriptor
#define FOR_TYPE(type, CALL)                                                                      \
    do {                                                                                          \
        if ((type) == ACH_F32) CALL(ACH_F32);                                                     \
        else if ((type) == ACH_BF16) CALL(ACH_BF16);                                              \
        else CALL(ACH_F16);                                                                       \
    } while (0)

extern "C" {

size_t ach_logprobs_workspace(const ach_logits_desc *desc, int k)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || k < 0 || k > ACH_TOP_MAX || k > d.classes) return 0;
    const Split s = split_rows(d.rows, d.classes);
    if (s.parts == 1) return 0;
    return (size_t)d.rows * s.parts * (sizeof(Total) + (size_t)k * sizeof(uint64_t));
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
    const size_t need = ach_logprobs_workspace(desc, k);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 16))) return ACH_EWORKSPACE;
    if (d.rows == 0) return ACH_OK;
    const Split sp = split_rows(d.rows, d.classes);
    const int nt = threads_for(sp.span, k);
    const dim3 grid(grid_of((size_t)d.rows * sp.parts));
    Total *part = (Total *)ws;
    uint64_t *lists = (uint64_t *)(part + (size_t)d.rows * sp.parts);
    const LogprobsOut o = {logprobs, ranks, entropy, stats, top_ids, top_logprobs};
    hipStream_t st = as_stream(s);
#define GO_(TYPE, NT, E, R)                                                                       \
    hipLaunchKernelGGL((k_logprobs<TYPE, NT, E, R>), grid, dim3(NT), 0, st, d,                    \
                       (const Elem<TYPE>::T *)logits, ids, k, o, sp.parts, sp.span, part, lists)
#define GO(TYPE, NT)                                                                              \
    do {                                                                                          \
        if (entropy && ranks) GO_(TYPE, NT, true, true);                                          \
        else if (entropy) GO_(TYPE, NT, true, false);                                             \
        else if (ranks) GO_(TYPE, NT, false, true);                                               \
        else GO_(TYPE, NT, false, false);                                                         \
    } while (0)
#define CALL(TYPE)                                                                                \
    do {                                                                                          \
        if (nt == 64) GO(TYPE, 64);                                                               \
        else if (nt == 256) GO(TYPE, 256);                                                        \
        else GO(TYPE, 1024);                                                                      \
    } while (0)
    FOR_TYPE(d.type, CALL);
#undef CALL
#undef GO
#undef GO_
    const int rc = check_launch();
    if (rc || sp.parts == 1) return rc;
#define CALL(TYPE)                                                                                \
    hipLaunchKernelGGL((k_logprobs_join<TYPE, 256>), dim3(grid_of(d.rows)), dim3(256), 0, st, d,  \
                       (const Elem<TYPE>::T *)logits, ids, k, o, sp.parts, part, lists)
    FOR_TYPE(d.type, CALL);
#undef CALL
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
    const int chunks = d.classes / (16 / (int)elem_size(d.type)), span = 1024;
    const int parts = chunks > span ? (chunks + span - 1) / span : 1;
    const dim3 grid(grid_of((size_t)d.rows * parts)), block(256);
    hipStream_t st = as_stream(s);
#define CALL(TYPE)                                                                                \
    hipLaunchKernelGGL((k_logprobs_bwd<TYPE>), grid, block, 0, st, d,                             \
                       (const Elem<TYPE>::T *)logits, ids, stats, entropy, dlogprobs, dentropy,   \
                       (Elem<TYPE>::T *)dlogits, dstride, parts, span)
    FOR_TYPE(d.type, CALL);
#undef CALL
    return check_launch();
}

// The workspace: the rows' losses, then, for rows in parts, the parts' sums
// and the rows' listed classes.
size_t ach_distill_workspace(const ach_logits_desc *desc, const ach_distill_desc *t)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || !distill_desc(t)) return 0;
    const Split s = split_rows(d.rows, d.classes);
    size_t n = round16((size_t)d.rows * sizeof(float));
    if (s.parts > 1)
        n += round16((size_t)d.rows * s.parts * sizeof(Dense)) +
             (size_t)d.rows * (ACH_TOP_MAX + 1) * sizeof(Entry);
    return n;
}

int ach_distill_xent(const ach_logits_desc *desc, const ach_distill_desc *teacher,
                     const void *logits, const int32_t *teacher_ids, const void *teacher_values,
                     const int32_t *labels, const float *row_weights, float *loss, void *delta,
                     int64_t delta_stride, float *cost, void *ws, size_t ws_bytes,
                     ach_stream_t s)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || !distill_desc(teacher)) return ACH_EINVAL;
    const ach_distill_desc t = *teacher;
    if (!logits || !aligned(logits, elem_size(d.type))) return ACH_EINVAL;
    if (!loss && !delta && !cost) return ACH_EINVAL;
    if (t.soft != 0.f && (!teacher_ids || !teacher_values)) return ACH_EINVAL;
    if (teacher_values && !aligned(teacher_values, elem_size(t.teacher_type))) return ACH_EINVAL;
    if (t.hard != 0.f && !labels) return ACH_EINVAL;
    if (!aligned(delta, elem_size(d.type))) return ACH_EINVAL;
    if (delta_stride == 0) delta_stride = d.classes;
    if (delta && (delta_stride < d.classes || (delta == logits && delta_stride != d.stride)))
        return ACH_EINVAL;
    const size_t need = ach_distill_workspace(desc, teacher);
    if (d.rows > 0 && (!ws || ws_bytes < need || !aligned(ws, 16))) return ACH_EWORKSPACE;
    hipStream_t st = as_stream(s);
    if (d.rows > 0) {
        const Split sp = split_rows(d.rows, d.classes);
        const int nt = threads_for(sp.span, 0);
        const bool two = t.soft != 0.f && t.hard != 0.f && d.temperature != 1.f;
        if (t.soft == 0.f) d.temperature = 1.f;  // the label's term is at temperature 1
        const dim3 grid(grid_of((size_t)d.rows * sp.parts));
        float *row_loss = (float *)ws;
        Dense *dense = (Dense *)((char *)ws + round16((size_t)d.rows * sizeof(float)));
        Entry *entries =
            (Entry *)((char *)dense + round16((size_t)d.rows * sp.parts * sizeof(Dense)));
#define GO(TYPE, NT, TWO, MODE)                                                                   \
    hipLaunchKernelGGL((k_distill<TYPE, NT, TWO, MODE>), grid, dim3(NT), 0, st, d, t,             \
                       (const Elem<TYPE>::T *)logits, teacher_ids, teacher_values, labels,        \
                       row_weights, loss, (Elem<TYPE>::T *)delta, delta_stride, row_loss,         \
                       sp.parts, sp.span, dense, entries)
#define WITH(TYPE, TWO)                                                                           \
    do {                                                                                          \
        if (sp.parts > 1) {                                                                       \
            if (nt == 256) GO(TYPE, 256, TWO, STATS);                                             \
            else GO(TYPE, 1024, TWO, STATS);                                                      \
            if (nt == 256) GO(TYPE, 256, TWO, DELTA);                                             \
            else GO(TYPE, 1024, TWO, DELTA);                                                      \
        } else if (nt == 64) GO(TYPE, 64, TWO, WHOLE);                                            \
        else if (nt == 256) GO(TYPE, 256, TWO, WHOLE);                                            \
        else GO(TYPE, 1024, TWO, WHOLE);                                                          \
    } while (0)
#define CALL(TYPE)                                                                                \
    do {                                                                                          \
        if (two) WITH(TYPE, true);                                                                \
        else WITH(TYPE, false);                                                                   \
    } while (0)
        FOR_TYPE(d.type, CALL);
#undef CALL
#undef WITH
#undef GO
        const int rc = check_launch();
        if (rc || !cost) return rc;
    }
    if (!cost) return ACH_OK;
    hipLaunchKernelGGL(k_sum_losses, dim3(1), dim3(256), 0, st, (const float *)ws, d.rows, cost);
    return check_launch();
}

}  // extern "C"
