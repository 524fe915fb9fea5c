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
#include "rows.hpp"

#include <float.h>
#include <math.h>

namespace ach {
namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// The elements of a chunk one after the other, in a loop that is not unrolled:
// what a workgroup does once per row costs more to fetch than to run.
template <int TYPE> struct Walk {
    static constexpr int VEC = Row<TYPE>::VEC;
    uint32_t w[4];
    __device__ explicit Walk(const typename Row<TYPE>::T *p)
    {
        const typename Row<TYPE>::Chunk v = Row<TYPE>::load(p);
        __builtin_memcpy(w, &v, 16);
    }
    __device__ __forceinline__ float next()
    {
        const uint32_t first = w[0];
        if (TYPE == ACH_F32) {
            w[0] = w[1], w[1] = w[2], w[2] = w[3];
            return __uint_as_float(first);
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) w[i] = w[i] >> 16 | w[i + 1] << 16;
        w[3] >>= 16;
        if (TYPE == ACH_BF16) return __uint_as_float(first << 16);
        const uint16_t half = (uint16_t)first;
        _Float16 h;
        __builtin_memcpy(&h, &half, 2);
        return (float)h;
    }
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

template <bool B> struct Flag {
    static constexpr bool value = B;
};

// Orders a wave's LDS accesses among its lanes.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
// sum for t a NaN, 0 * -inf: then it is formed again without them.  Returns the
// lane's maximum of them.
template <bool FULL, int N>
__device__ __forceinline__ float absorb(Stat &a, const float (&x)[N], float c, float x_id)
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
        if (FULL) t = fmaf(e, d, t);
        if (FULL) a.above += __popcll(__ballot(x[i] > x_id));
    }
    if (FULL) {
        if (t != t) {
            t = a.t;
            for (int i = 0; i < N; ++i) {
                const float d = fmaxf((x[i] - a.m) * c, FAR);
                t = fmaf(exp2_fast(d), d, t);
            }
        }
        a.t = t;
    }
    return m;
}

// How a range's chunks are read: `full` times UNROLL chunks by every thread,
// chunk q by thread q % NT, then what is left.  With alternatives to be found,
// the maxima of what a thread reads in 2^shift turns, a group, and of what is
// left are kept.
constexpr int UNROLL = 4;
constexpr int groups_of(int threads) { return threads == 64 ? 8 : 16; }

template <int TYPE, int NT> struct Turns {
    static constexpr int GROUPS = groups_of(NT);
    int full, shift;
    __device__ explicit Turns(const Range<TYPE> &g)
        : full(g.chunks() / (UNROLL * NT)), shift(0)
    {
        while (full > GROUPS << shift) ++shift;
    }
    // chunk i of a thread's group, or -1
    __device__ int chunk(const Range<TYPE> &g, int group, int thread, int i) const
    {
        const int turn = group == GROUPS ? full : (group << shift) + i / UNROLL;
        if (group == GROUPS ? i >= UNROLL : turn >= full) return -1;
        const int q = (turn * UNROLL + i % UNROLL) * NT + thread;
        return q < g.chunks() ? q : -1;
    }
};

template <int NT> struct GroupLds {
    float most[groups_of(NT) + 1][NT];
};

template <int TYPE, int NT, bool FULL, bool TOP>
__device__ __forceinline__ Stat stream(const Range<TYPE> &g, const Turns<TYPE, NT> &turns, float c,
                                       float x_id, GroupLds<NT> *groups)
{
    constexpr int V = Row<TYPE>::VEC, U = UNROLL;
    typedef typename Row<TYPE>::Chunk Chunk;
    Stat a = {-FLT_MAX, 0.f, 0.f, 0};
    const int n = g.chunks(), lane = threadIdx.x & 63;
    const auto *p = g.p + (size_t)threadIdx.x * V;
    float most = -INFINITY;
    for (int turn = 0; turn < turns.full; ++turn, p += (size_t)U * NT * V) {
        Chunk v[U];
        float x[U * V];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = Row<TYPE>::load(p + (size_t)u * NT * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) x[u * V + i] = (float)v[u][i];
        const float m = absorb<FULL>(a, x, c, x_id);
        if (TOP) {
            most = fmaxf(most, m);
            if (((turn + 1) & ((1 << turns.shift) - 1)) == 0 || turn + 1 == turns.full) {
                groups->most[turn >> turns.shift][threadIdx.x] = most;
                most = -INFINITY;
            }
        }
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63);
    const int left = turns.full * U * NT + wave;  // fewer than U turns of one chunk
    Chunk v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (left + u * NT + lane < n)
            v[u] = Row<TYPE>::load(g.p + (size_t)(left + u * NT + lane) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (left + u * NT >= n) break;
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = left + u * NT + lane < n ? (float)v[u][i] : -INFINITY;
        most = fmaxf(most, absorb<FULL>(a, x, c, x_id));
    }
    if (wave == 0) {
        const float x[1] = {lane < g.rest() ? (float)g.p[(size_t)n * V + lane] : -INFINITY};
        most = fmaxf(most, absorb<FULL>(a, x, c, x_id));
    }
    if (TOP) groups->most[groups_of(NT)][threadIdx.x] = most;
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
// these.  Only groups whose maximum reaches that bound hold candidates, so only
// they are read again (from the caches), by all threads together.  Of random
// logits some k log(waves) + k pass; they are put in order by counting for each
// how many are before it.
template <int NT> struct TopLds {
    // logits above the bound, and at it; groups to be read again
    static constexpr int CAP = NT == 64 ? 256 : 1024, EQUAL = NT == 64 ? 128 : 512,
                         HOT = NT == 64 ? 128 : 512, GROUPS = groups_of(NT);
    alignas(16) uint64_t list[CAP + EQUAL + 8];
    uint64_t equal[EQUAL];
    GroupLds<NT> groups;
    uint32_t bound[NT / 64];
    int hot[HOT];
    int sum[NT / 64], places[64];
    int nhot, nlist, nequal;
};

// f(x, class) for every logit of the groups whose maximum reaches `low`,
// which are listed unless they are too many, and the single elements.  Of groups
// that are not listed, those are left out of whose maximum skip() says so.
template <int TYPE, int NT, class F, class S>
__device__ __forceinline__ void each_hot(const Range<TYPE> &g, const Turns<TYPE, NT> &turns,
                                         const TopLds<NT> &sh, float low, S skip, F f)
{
    constexpr int V = Row<TYPE>::VEC, GROUPS = groups_of(NT);
    const auto chunk = [&](int q) {
        if (q < 0) return;
        Walk<TYPE> walk(g.p + (size_t)q * V);
#pragma unroll 1
        for (int e = 0; e < V; ++e) f(walk.next(), g.begin + q * V + e);
    };
    const int each = UNROLL << turns.shift;
    if (sh.nhot <= TopLds<NT>::HOT) {
        for (int i = threadIdx.x; i < sh.nhot * each; i += NT) {
            const int h = sh.hot[i / UNROLL >> turns.shift];
            chunk(turns.chunk(g, h / NT, h % NT, i & (each - 1)));
        }
    } else {
        for (int group = 0; group <= GROUPS; ++group)
            if (group == GROUPS || (group << turns.shift) < turns.full)
                if (const float most = sh.groups.most[group][threadIdx.x];
                    most >= low && !skip(most))
                    for (int i = 0; i < each; ++i)
                        chunk(turns.chunk(g, group, threadIdx.x, i));
    }
    if (threadIdx.x < g.rest()) {
        const int j = g.chunks() * V + threadIdx.x;
        f((float)g.p[j], g.begin + j);
    }
}

// The upper 16 bits of the nth largest key of the wave's lanes: a lower bound,
// 0 if there are not so many lanes.
__device__ __forceinline__ uint32_t nth_largest(uint32_t key, int nth)
{
    uint32_t bound = 0;
#pragma unroll 1
    for (int b = 31; b >= 16; --b) {
        const uint32_t up = bound | 1u << b;
        if (__popcll(__ballot(key >= up)) >= nth) bound = up;
    }
    return bound;
}

// Leaves in sh.list a superset of the k largest of the range (k <= its
// length, no NaN) and returns its size; `mine` is the thread's maximum.
template <int TYPE, int NT>
__device__ __forceinline__ int candidates(const Range<TYPE> &g, const Turns<TYPE, NT> &turns,
                                          float mine, int k, TopLds<NT> &sh)
{
    constexpr int CAP = TopLds<NT>::CAP, EQUAL = TopLds<NT>::EQUAL, W = NT / 64;
    constexpr int GROUPS = groups_of(NT);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nth = (k + W - 1) / W;
    const uint32_t key = order_key(mine);
    uint32_t bound = nth_largest(key, nth);
    __syncthreads();
    if (lane == 0) sh.bound[wave] = bound;
    if (threadIdx.x == 0) sh.nhot = sh.nlist = sh.nequal = 0;
    __syncthreads();
    for (int i = 0; i < W; ++i) bound = min(bound, sh.bound[i]);
    // up to -FLT_MAX, where a thread that has seen -inf alone starts: anything
    float low = bound <= order_key(-FLT_MAX) ? -INFINITY : key_value(bound);
    // (logits of -inf are no candidates: the last loop takes those that are wanted)
    const float first_low = fmaxf(low, -FLT_MAX);
    if (mine >= first_low) {
        const int groups = (turns.full + (1 << turns.shift) - 1) >> turns.shift;
        for (int i = 0; i <= groups; ++i) {
            const int group = i < groups ? i : GROUPS;
            if (sh.groups.most[group][threadIdx.x] < first_low) continue;
            const int to = atomicAdd(&sh.nhot, 1);
            if (to < TopLds<NT>::HOT) sh.hot[to] = group * NT + threadIdx.x;
        }
    }
    __syncthreads();
    while (true) {
        // Once there are more equal logits than there is room for, their number
        // does not matter, and a group that holds nothing larger is not read:
        // 72 us for 1024 rows of 131072 equal bf16 logits, 482 if all are counted.
        const auto skip = [&](float most) {
            return most <= low && *(volatile int *)&sh.nequal > EQUAL;
        };
        each_hot<TYPE, NT>(g, turns, sh, first_low, skip, [&](float x, int j) {
            if (!(x >= low) || x == -INFINITY) return;
            const bool above = x > low;
            const int i = atomicAdd(above ? &sh.nlist : &sh.nequal, 1);
            if (i < (above ? CAP : EQUAL)) (above ? sh.list : sh.equal)[i] = compound(x, j);
        });
        __syncthreads();
        if (sh.nlist <= CAP) break;
        // Too many: the k-th largest itself, bit by bit.  No logits are above
        // it that are not among the k, so the next round is the last.
        uint32_t kth = 0;
        for (int b = 31; b >= 0; --b) {
            const uint32_t up = kth | (1u << b);
            int count = 0;
            each_hot<TYPE, NT>(g, turns, sh, first_low, [](float) { return false; },
                               [&](float x, int) { count += order_key(x) >= up; });
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

// emit(place, compound) for the k largest of list[0..n), largest first, by
// counting for each how many are before it.  The list is filled up with zeros,
// which no logit's compound is below, to a multiple of 8 (there has to be
// room).  Up to 64 are counted by all waves together, each against its share.
__device__ __forceinline__ int count_larger(const uint64_t *list, int from, int to, uint64_t v)
{
    int n = 0;
    for (int j = from; j < to; j += 8) {
        uint64_t w[8];
#pragma unroll
        for (int l = 0; l < 8; ++l) w[l] = list[j + l];
#pragma unroll
        for (int l = 0; l < 8; ++l) n += w[l] > v;
    }
    return n;
}

template <int NT, class F>
__device__ __forceinline__ void in_order(uint64_t *list, int n, int k, int *places, F emit)
{
    const int n8 = (n + 7) & ~7, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)threadIdx.x < n8 - n) list[n + threadIdx.x] = 0;
    if (NT > 64 && n <= 64) {
        if (wave == 0) places[lane] = 0;
        __syncthreads();
        const uint64_t v = lane < n ? list[lane] : 0;
        const int share = (n8 / 8 + NT / 64 - 1) / (NT / 64) * 8, from = wave * share;
        if (from < n8 && lane < n)
            atomicAdd(&places[lane], count_larger(list, from, min(from + share, n8), v));
        __syncthreads();
        if (wave == 0 && lane < n && places[lane] < k) emit(places[lane], v);
        return;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t v = list[i];
        const int place = count_larger(list, 0, n8, v);
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

// (x - m)/T, also where the difference is beyond the largest number of 32 bits,
// as for masks of a type's lowest value, and its quotient is not.
__device__ __forceinline__ float scaled(float x, float m, float inv_t)
{
    return (float)(((double)x - m) * inv_t);
}

// A row's outputs but its alternatives; returns the log of its sum.
__device__ float write_row(const LogprobsOut &o, int r, const Total &a, bool given, float x_id,
                           float inv_t, bool first_thread)
{
    const bool bad = !(a.rest < INFINITY), empty = a.m == -INFINITY && !bad;
    const float log_s = empty ? -INFINITY : log1pf(a.rest);
    if (first_thread) {
        if (o.logprobs)
            o.logprobs[r] = !given ? 0.f : empty ? -INFINITY : scaled(x_id, a.m, inv_t) - log_s;
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
        m == -INFINITY ? -INFINITY : scaled(key_value((uint32_t)(v >> 32)), m, inv_t) - log_s;
}

template <bool B, class X, class Y> struct Pick {
    using T = X;
};
template <class X, class Y> struct Pick<false, X, Y> {
    using T = Y;
};

// One workgroup per row, or per part of a row (parts > 1), `span` classes
// each; the parts' totals and their k largest go to `part` and `lists`.
// 4096 x 32768 bf16 without alternatives: 55 us, 4.9 TB/s, the vector unit 85%
// busy with 11 instructions a logit.  1024 x 131072 bf16 with 20: 59 us, 4.5 TB/s;
// its rows are all in step, so the 4 us of the alternatives show.
template <int TYPE, int NT, bool FULL, bool TOP>
__global__ void __launch_bounds__(NT)
    k_logprobs(ach_logits_desc d, const typename Elem<TYPE>::T *__restrict__ logits,
               const int32_t *__restrict__ ids, int k, LogprobsOut o, int parts, int span,
               Total *__restrict__ part, uint64_t *__restrict__ lists)
{
    __shared__ StatLds<NT> st;
    __shared__ typename Pick<TOP, TopLds<NT>, char>::T top;
    const float inv_t = 1.f / d.temperature, c = inv_t * LOG2E;
    for (size_t w = blockIdx.x; w < (size_t)d.rows * parts; w += gridDim.x) {
        const int r = (int)(w / parts), at = (int)(w % parts) * span;
        const auto *row = logits + (size_t)r * d.stride;
        const Range<TYPE> g = {row + at, at, min(span, d.classes - at)};
        const int id = ids ? ids[r] : -1;
        const bool given = id >= 0 && id < d.classes;
        const float x_id = given ? (float)row[id] : INFINITY;
        const Turns<TYPE, NT> turns(g);
        GroupLds<NT> *groups = nullptr;
        if constexpr (TOP) groups = &top.groups;
        const Stat mine = stream<TYPE, NT, FULL, TOP>(g, turns, c, x_id, groups);
        const Total a = total_of<TYPE, NT>(g, mine, c, st);
        if (parts > 1 && threadIdx.x == 0) part[w] = a;
        const float log_s = parts > 1 ? 0.f
                                      : write_row(o, r, a, given, x_id, inv_t, threadIdx.x == 0);
        if constexpr (TOP) {
            if (!(a.rest < INFINITY)) {  // a NaN or a +inf: the join sees it in the total
                for (int i = threadIdx.x; i < k && parts == 1; i += NT) {
                    o.top_ids[(size_t)r * k + i] = -1;
                    o.top_logprobs[(size_t)r * k + i] = NAN;
                }
            } else {
                const int mk = min(k, g.len), n = candidates<TYPE, NT>(g, turns, mine.m, mk, top);
                in_order<NT>(top.list, n, mk, top.places, [&](int i, uint64_t v) {
                    if (parts > 1) lists[w * k + i] = v;
                    else write_top(o, (size_t)r * k + i, v, a.m, inv_t, log_s);
                });
                if (parts > 1)
                    for (int i = mk + threadIdx.x; i < k; i += NT) lists[w * k + i] = 0;
            }
        }
        __syncthreads();
    }
}

// Joins the parts of a row.  Of the parts' lists, for every m the m-th largest
// of their ceil(k/m)-th entries bounds the k-th largest of all from below: one
// part may hold the largest, or all parts evenly.  Entries that pass the best
// of four such bounds, of 16 bits, are put in order.  If these are many,
// logits being equal or spread unevenly, the same bounds are taken exactly and
// for every power of two: then, for m = 1, 2, 4, ..., no more than m lists have
// ceil(k/m) entries that pass, which adds up to k (2 + log2 parts).  A chain of
// waits: 5 us for one row of 32 parts with 20 entries each.
constexpr int MOST_PARTS = 64;

template <int TYPE, int NT>
__global__ void __launch_bounds__(NT)
    k_logprobs_join(ach_logits_desc d, const typename Elem<TYPE>::T *__restrict__ logits,
                    const int32_t *__restrict__ ids, int k, LogprobsOut o, int parts,
                    const Total *__restrict__ part, const uint64_t *__restrict__ lists)
{
    constexpr int STAGE = 2048, CAP = ACH_TOP_MAX * 8, W = NT / 64;
    // Times k; of random logits some 2 k pass.  One row of 131072 equal bf16
    // logits, k = 20: 20 us, and 41 if only what does not fit is narrowed down.
    constexpr int MANY = 4;
    static_assert(W == 4 && CAP >= ACH_TOP_MAX * 8, "four bounds; room for the exact ones");
    static_assert(CAP > MANY * ACH_TOP_MAX, "an overflow is many");
    const float inv_t = 1.f / d.temperature, c = inv_t * LOG2E;
    alignas(16) __shared__ uint64_t list[CAP + 8];
    __shared__ uint64_t stage[STAGE], bounds[8], nth_of[W][64];
    __shared__ int n, places[64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = blockIdx.x; r < d.rows; r += gridDim.x) {
        const int id = ids ? ids[r] : -1;
        // the lists, where they fit, to be read from LDS
        const uint64_t *from = lists + (size_t)r * parts * k;
        const int entries = parts * k;
        const bool staged = entries <= STAGE;
        uint64_t staging[STAGE / NT];
        if (staged)
#pragma unroll
            for (int i = 0; i < STAGE / NT; ++i)
                if ((int)threadIdx.x + i * NT < entries) staging[i] = from[threadIdx.x + i * NT];
        Total a = {-INFINITY, 0.f, 0.f, 0};
        if (lane < parts) a = part[(size_t)r * parts + lane];
        const bool given = id >= 0 && id < d.classes;
        const float x_id = given ? (float)logits[(size_t)r * d.stride + id] : 0.f;
        __syncthreads();  // of the last row
        if (staged)
#pragma unroll
            for (int i = 0; i < STAGE / NT; ++i)
                if ((int)threadIdx.x + i * NT < entries) stage[threadIdx.x + i * NT] = staging[i];
        if (threadIdx.x == 0) n = 0;
        const auto entry = [&](int i) { return staged ? stage[i] : from[i]; };
        // every wave joins the totals by itself
        const bool bad = __any(!(a.rest < INFINITY));
        const float m = wave_most(a.m);
        const uint64_t at_max = __ballot(a.m == m && lane < parts);
        const int owner = at_max ? __ffsll((unsigned long long)at_max) - 1 : 0;
        const float z = m == -INFINITY ? 0.f : fmaxf((a.m - m) * c, FAR);
        const float f = a.m == -INFINITY ? 0.f : exp2_fast(z), s = 1.f + a.rest;
        Total t;
        t.m = m;
        t.rest = wave_total(a.m == -INFINITY ? 0.f : lane == owner ? a.rest : s * f);
        if (bad) t.rest = NAN;
        t.t = wave_total(a.m == -INFINITY ? 0.f : f * (a.t + s * z));
        t.above = wave_all(a.above, Add());
        const float log_s = write_row(o, r, t, given, x_id, inv_t, threadIdx.x == 0);
        if (k == 0) continue;
        if (bad) {
            for (int i = threadIdx.x; i < k; i += NT) {
                o.top_ids[(size_t)r * k + i] = -1;
                o.top_logprobs[(size_t)r * k + i] = NAN;
            }
            continue;
        }
        __syncthreads();
        uint64_t low = 1;  // 0 fills up short lists
        {
            int most = 1;
            while (most * 2 <= parts) most *= 2;
            const int of[4] = {1, 4, 16, most}, mine = min(of[wave], most);
            const int nth = (k + mine - 1) / mine;
            const uint64_t v = lane < parts ? entry(lane * k + nth - 1) : 0;
            const uint64_t bound = (uint64_t)nth_largest((uint32_t)(v >> 32), mine) << 32;
            if (lane == 0) bounds[wave] = bound;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) low = max(low, bounds[i]);
        const auto collect = [&] {
            for (int i = threadIdx.x; i < entries; i += NT) {
                const uint64_t v = entry(i);
                if (v < low) continue;
                const int to = atomicAdd(&n, 1);
                if (to < CAP) list[to] = v;
            }
            __syncthreads();
        };
        collect();
        if (n > MANY * k) {
            __syncthreads();
            if (threadIdx.x < 8) bounds[threadIdx.x] = 0;
            if (threadIdx.x == 0) n = 0;
            __syncthreads();
            for (int b = wave; b < 7 && (1 << b) <= parts; b += W) {
                const int nth = (k + (1 << b) - 1) >> b;
                const uint64_t v = lane < parts ? entry(lane * k + nth - 1) : 0;
                nth_of[wave][lane] = v;
                wave_sync();
                int before = 0;
                for (int i = 0; i < parts; ++i) {
                    const uint64_t other = nth_of[wave][i];
                    before += other > v || (other == v && i < lane);
                }
                wave_sync();
                if (lane < parts && before == (1 << b) - 1) bounds[b] = v;
            }
            __syncthreads();
            low = 1;
            for (int b = 0; b < 7; ++b) low = max(low, bounds[b]);
            collect();
        }
        in_order<NT>(list, min(n, CAP), k, places, [&](int i, uint64_t v) {
            write_top(o, (size_t)r * k + i, v, m, inv_t, log_s);
        });
    }
}

// Each workgroup writes `span` chunks of a row.  With l = log p,
// dx = p (a + b l) for a = -(g + h H)/T, b = -h/T; of the given class
// g (1 - p) = -g expm1(l), which keeps its precision where p is near 1.
// 4096 x 32768 bf16: 93 us, 5.7 TB/s.
template <int TYPE>
__global__ void __launch_bounds__(256)
    k_logprobs_bwd(ach_logits_desc d, const typename Elem<TYPE>::T *logits,
                   const int32_t *__restrict__ ids, const float *__restrict__ stats,
                   const float *__restrict__ entropy, const float *__restrict__ dlogprobs,
                   const float *__restrict__ dentropy, typename Elem<TYPE>::T *dlogits,
                   int64_t dstride, int parts, int span, bool past)
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
        const auto write = [&](auto PAST) {
            for (int q = first + threadIdx.x; q < last; q += 256) {
                Chunk v = {};
                if (!none) {
                    const Chunk x = Row<TYPE>::load(row + (size_t)q * V);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = (T)grad((float)x[i], q * V + i);
                }
                Row<TYPE>::template store<PAST.value>(out + (size_t)q * V, v);
            }
        };
        if (past) write(Flag<true>());
        else write(Flag<false>());
        if (last == chunks && threadIdx.x < rest) {
            const int j = chunks * V + threadIdx.x;
            out[j] = none ? (T)0.f : (T)grad((float)row[j], j);
        }
    }
}

// ---- distillation ------------------------------------------------------------------
// A row's listed classes, the teacher's entries and the label, are few, and
// their terms are formed one by one, sums of them in 64 bits.  All others, the
// dense ones, enter through their maximum and their sums of exponentials
// alone, so the sum over what the teacher leaves out is a sum of these, not a
// difference of nearly equal sums.  With e_j = exp((x_j - mo)/T) relative to
// the maximum mo of the dense classes, the delta of such a class is
// K e_j + K1 e1_j (e1: at temperature 1), and that of a listed one is written
// over it afterwards.
struct Dense {
    float m, s, s1;
};

// Whether the label's exponentials, at temperature 1, are wanted next to the
// teacher's, and how they are had: not apart (ONE), on their own, or at
// temperatures 2 and 4, which are common, as the second and fourth powers of
// these.  On their own and as powers: 2048 x 32768 bf16 72.3 and 67.2 us at
// temperature 2, 72.7 and 67.7 at 4; 4096 x 1000 fp32 17.9 and 17.3, 18.0 and
// 17.7; 1021 x 50021 fp16 62.0 and 61.1 at 2, fp32 no difference.
enum { ONE = 0, BOTH = 1, SQUARE = 2, FOURTH = 4 };

template <int TWO> __device__ __forceinline__ float second(float e, float d)
{
    if (TWO == BOTH) return exp2_fast(d * LOG2E);
    const float e2 = e * e;
    return TWO == SQUARE ? e2 : e2 * e2;
}

template <int TWO>
__device__ __forceinline__ void raise_dense(Dense &a, float m, float c)
{
    a.s *= exp2_fast(fmaxf((a.m - m) * c, FAR));
    if (TWO) a.s1 *= exp2_fast(fmaxf((a.m - m) * LOG2E, FAR));
    a.m = m;
}

// N logits, unless they are to be left out.
template <int TWO, int N>
__device__ __forceinline__ void absorb_dense(Dense &a, const float (&x)[N], float c, bool out)
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
    if (m > a.m && !out) raise_dense<TWO>(a, m, c);
    float s = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = x[i] - a.m, e = exp2_fast(d * c);
        s += e;
        if (TWO) s1 += second<TWO>(e, d);
    }
    a.s += out ? 0.f : s;
    if (TWO) a.s1 += out ? 0.f : s1;
}

// A wave's listed classes (classes 64 w to 64 w + 63 of the list): their
// maximum `most` (-inf if none is listed; 0 if none of them is finite: then e is
// 0, and `most` says nothing of where the row's logits lie) and that of the
// teacher's values, and relative to these the sums of e, e1, p, and
// p (log p - (x - most)/T).
struct Listed {
    float most, most_value;
    double e, e1, p, l;
};
constexpr int LISTED_WAVES = (ACH_TOP_MAX + 1 + 63) / 64;

// One listed class: relative to its wave's maxima.
struct Entry {
    int id;  // -1: none
    float e, e1, p;
};

template <int NT> struct DistillLds {
    uint32_t bits[NT + 1];      // the listed ones among the classes behind the last turn
    uint32_t dirty[NT];         // by thread: the turns that read a listed class
    // these, in a table by turn * NT + thread (-1: free), with a bit for each of
    // the turn's logits that is listed
    static constexpr int SLOTS = 256;
    int turn[SLOTS];
    uint32_t listed_bits[SLOTS];
    int owner[SLOTS];           // the first listed class that has it
    int slot[ACH_TOP_MAX + 1];  // by listed class; -1: none
    alignas(16) int id[ACH_TOP_MAX + 4];  // as they are given, the label at [k]; -1: none
    int repeated[ACH_TOP_MAX + 1];
    Dense wave[NT / 64];
    Listed listed[LISTED_WAVES];
    float x_y;                  // the label's logit
    int extra;                  // the label is a class that the teacher does not list
};

// Marks the listed classes of a range: the turns that read them, and of the
// classes behind the last turn each one.  Starts and ends with a barrier.
template <int TYPE, int NT>
__device__ __forceinline__ void mark(const Range<TYPE> &g, int k, int full, DistillLds<NT> &sh)
{
    constexpr int V = Row<TYPE>::VEC, U = UNROLL;
    static_assert(U * V <= 32, "the classes behind the last turn have their bits");
    __syncthreads();
    for (int i = threadIdx.x; i <= NT; i += NT) sh.bits[i] = 0;
    sh.dirty[threadIdx.x] = 0;
    constexpr int SLOTS = DistillLds<NT>::SLOTS;
    static_assert(SLOTS > ACH_TOP_MAX + 1, "a slot is always free");
    for (int i = threadIdx.x; i < SLOTS; i += NT) {
        sh.turn[i] = -1;
        sh.listed_bits[i] = 0;
        sh.owner[i] = ACH_TOP_MAX + 1;
    }
    __syncthreads();
    const int left = full * U * NT * V;
    for (int i = threadIdx.x; i <= k; i += NT) {
        const int j = sh.id[i] - g.begin;
        sh.slot[i] = -1;
        if (j < 0 || j >= g.len) continue;
        if (j >= left) {
            atomicOr(&sh.bits[(j - left) >> 5], 1u << ((j - left) & 31));
            continue;
        }
        const int q = j / V, turn = q / (U * NT), thread = q % NT, key = turn * NT + thread;
        atomicOr(&sh.dirty[thread], 1u << turn);
        int slot = (thread + 61 * turn) % SLOTS;
        while (true) {
            const int old = atomicCAS(&sh.turn[slot], -1, key);
            if (old == -1 || old == key) break;
            slot = (slot + 1) % SLOTS;
        }
        sh.slot[i] = slot;
        atomicMin(&sh.owner[slot], i);
        atomicOr(&sh.listed_bits[slot], 1u << (q / NT % U * V + j % V));
    }
    __syncthreads();
}

// The chunks of the marked turns, the chunks behind the last turn and the
// single elements, with the listed classes masked.
template <int TYPE, int NT, int TWO>
__device__ __forceinline__ void absorb_masked(Dense &a, const Range<TYPE> &g, float c, int k,
                                              int full, const DistillLds<NT> &sh)
{
    constexpr int V = Row<TYPE>::VEC, U = UNROLL;
    const auto absorb = [&](const typename Row<TYPE>::Chunk &v, uint32_t mask) {
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = mask >> e & 1 ? -INFINITY : (float)v[e];
        absorb_dense<TWO>(a, x, c, false);
    };
    // a turn by the first of its listed classes, so that the sums have one order
    for (int i = threadIdx.x; i < (k + 1) * U; i += NT) {
        const int slot = sh.slot[i / U];
        if (slot < 0 || sh.owner[slot] != i / U) continue;
        const int turn = sh.turn[slot];
        const int q = (turn / NT * U + i % U) * NT + turn % NT;
        absorb(Row<TYPE>::load(g.p + (size_t)q * V), sh.listed_bits[slot] >> (i % U * V));
    }
    const int n = g.chunks(), left = full * U * NT;
    typename Row<TYPE>::Chunk v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int q = left + u * NT + threadIdx.x;
        if (q < n) v[u] = Row<TYPE>::load(g.p + (size_t)q * V);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int q = u * NT + threadIdx.x;
        if (left + q >= n) break;
        absorb(v[u], sh.bits[q * V >> 5] >> (q * V & 31));
    }
    if (threadIdx.x < g.rest()) {
        const int j = n * V + threadIdx.x, b = j - left * V;
        const float x[1] = {sh.bits[b >> 5] >> (b & 31) & 1 ? -INFINITY : (float)g.p[j]};
        absorb_dense<TWO>(a, x, c, false);
    }
}

// A thread's statistics of the dense classes of a range.  A turn that reads a
// listed class is left out (by the one thread), and its chunks are read again
// with the listed classes masked.  The first `stashed` turns stay in LDS.
template <int TYPE, int NT, int TWO>
__device__ __forceinline__ Dense stream_dense(const Range<TYPE> &all, float c, int k, int stashed,
                                              DistillLds<NT> &sh)
{
    constexpr int V = Row<TYPE>::VEC, U = UNROLL, SEG = 32 * U * V * NT;  // 32 turns
    typedef typename Row<TYPE>::Chunk Chunk;
    extern __shared__ uint4 stash[];
    Dense a = {-FLT_MAX, 0.f, 0.f};
    for (int at = 0; at < all.len; at += SEG) {
        const Range<TYPE> g = {all.p + at, all.begin + at, min(SEG, all.len - at)};
        const int full = g.chunks() / (U * NT);
        mark<TYPE, NT>(g, k, full, sh);
        uint32_t dirty = sh.dirty[threadIdx.x];
        const auto *p = g.p + (size_t)threadIdx.x * V;
        for (int turn = 0; turn < full; ++turn, dirty >>= 1, p += (size_t)U * NT * V) {
            Chunk v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = Row<TYPE>::load(p + (size_t)u * NT * V);
            if (at == 0 && turn < stashed)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    __builtin_memcpy(&stash[(turn * U + u) * NT + threadIdx.x], &v[u], 16);
            float x[U * V];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) x[u * V + i] = (float)v[u][i];
            absorb_dense<TWO>(a, x, c, dirty & 1);
        }
        absorb_masked<TYPE, NT, TWO>(a, g, c, k, full, sh);
    }
    return a;
}

// The same of the wave, in all its lanes.
template <int TWO> __device__ __forceinline__ void wave_dense(Dense &a, float c)
{
    raise_dense<TWO>(a, wave_most(a.m), c);
    a.s = wave_total(a.s);
    if (TWO) a.s1 = wave_total(a.s1);
}

__device__ __forceinline__ float load_any(const void *p, int type, size_t i)
{
    return type == ACH_F32    ? ((const float *)p)[i]
           : type == ACH_BF16 ? (float)((const __bf16 *)p)[i]
                              : (float)((const _Float16 *)p)[i];
}

// Marks the listed classes that an earlier one of the list equals: the threads
// that share a class each look through a part of the list, four at a time.
template <int NT> __device__ __forceinline__ void find_repeated(int k, DistillLds<NT> &sh)
{
    int shift = 0;
    while (1 << shift <= k) ++shift;
    const int later = threadIdx.x & ((1 << shift) - 1), share = threadIdx.x >> shift;
    if (later > k) return;
    const int id = sh.id[later], step = 4 * (NT >> shift);
    bool found = false;
    for (int i = 4 * share; i < later; i += step)
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= sh.id[i + j] == id && i + j < later;
    if (found) sh.repeated[later] = 1;
}

// The listed classes of a row, k + 1 <= NT.  Class i of the list is thread i's
// `entry`; the waves' sums are left in sh.listed.  sh.id and sh.repeated have
// been filled in, and a barrier has been since.
template <int TYPE, int NT, int TWO>
__device__ __forceinline__ void listed_terms(Entry &entry, const typename Elem<TYPE>::T *row,
                                             const void *values, int type, size_t at, int k,
                                             bool tail, float temperature, double inv_td,
                                             DistillLds<NT> &sh)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = threadIdx.x;
    const float inv_t = 1.f / temperature, c = inv_t * LOG2E;
    entry = {-1, 0.f, 0.f, 0.f};
    if (wave > k >> 6) return;  // no class of this wave is listed
    Listed sum = {-INFINITY, -INFINITY, 0, 0, 0, 0};
    float x = -INFINITY, value = -INFINITY;
    const int id = i <= k ? sh.id[i] : -1;
    if (id >= 0) {
        x = (float)row[id];
        if (i < k) value = load_any(values, type, at + i);
        else sh.x_y = x;
        // of entries with the same id the first counts; the label, at [k], is last
        if (!sh.repeated[i]) entry.id = id;
        else x = value = -INFINITY;
    }
    sum.most = wave_most(x);
    sum.most_value = wave_most(value);
    if (sum.most == -INFINITY && __any(id >= 0)) sum.most = 0.f;
    if (entry.id >= 0) {
        entry.e = exp2_fast((x - sum.most) * c);
        entry.e1 = TWO ? exp2_fast((x - sum.most) * LOG2E) : entry.e;
        sum.e = entry.e;
        sum.e1 = entry.e1;
        if (value != -INFINITY) {
            const double l = tail ? (double)value : ((double)value - sum.most_value) * inv_td;
            sum.p = exp(l);
            entry.p = (float)sum.p;
            if (sum.p != 0) sum.l = sum.p * (l - ((double)x - sum.most) * inv_td);
        }
    }
    sum.e = wave_total(sum.e);
    sum.e1 = wave_total(sum.e1);
    sum.p = wave_total(sum.p);
    sum.l = wave_total(sum.l);
    if (lane == 63) sh.listed[wave] = sum;
}

// What the delta and the loss of a row are made of.
struct RowTerms {
    float m;              // of the dense classes
    float K, K1;          // their factors
    float P_total, one_total, soft, hard, scale, y_rest;
    float to_e[LISTED_WAVES], to_e1[LISTED_WAVES], to_p[LISTED_WAVES];  // from a wave's maxima
    float loss;
    bool empty, none;  // no logit, or no listed class: all of it is 0
};

template <int TWO>
__device__ __forceinline__ RowTerms row_terms(const Dense &a, const Listed *listed, int waves,
                                              const ach_distill_desc &t, int k, float temperature,
                                              bool label, bool extra, float x_y, float w)
{
    const bool tail = t.mode == ACH_DISTILL_TAIL;
    const float c = LOG2E / temperature;
    const double inv_td = 1. / temperature;
    RowTerms o;
    o.m = a.m;
    float ref = a.m, most_value = -INFINITY;  // the row's maximum
    o.none = true;
    for (int i = 0; i < waves; ++i) {
        o.none &= listed[i].most == -INFINITY;
        if (listed[i].e != 0) ref = fmaxf(ref, listed[i].most);
        most_value = fmaxf(most_value, listed[i].most_value);
    }
    double e = 0, e1 = 0, p = 0, l = 0;
#pragma unroll
    for (int i = 0; i < LISTED_WAVES; ++i) {
        o.to_e[i] = o.to_e1[i] = o.to_p[i] = 0.f;
        if (i >= waves) continue;
        const Listed &s = listed[i];
        // where a wave's classes are all masked the factors stay 0: from `most` they
        // would be infinite in rows of low logits, and 0 times that a NaN
        if (s.e != 0) {
            o.to_e[i] = exp2_fast((s.most - ref) * c);
            o.to_e1[i] = TWO ? exp2_fast((s.most - ref) * LOG2E) : o.to_e[i];
            e += s.e * o.to_e[i];
            e1 += s.e1 * o.to_e1[i];
        }
        // in 64 bits: a class that the student has masked makes s.l infinite,
        // however little probability the teacher gives it
        const double lower =
            tail || s.most_value == -INFINITY ? 0 : (double)s.most_value - most_value;
        const double to_p = lower == 0 ? 1 : exp(lower * inv_td);
        o.to_p[i] = (float)to_p;
        if (s.p == 0 || to_p == 0) continue;
        p += s.p * to_p;
        l += to_p * (s.l + s.p * (lower - ((double)s.most - ref)) * inv_td);
    }
    // without a dense class of finite logit a.s is 0
    const float up = exp2_fast((a.m - ref) * c), up1 = TWO ? exp2_fast((a.m - ref) * LOG2E) : up;
    const double total = e + (double)a.s * up, total1 = e1 + (double)a.s1 * up1;
    o.empty = total == 0;
    // the largest logit counts exactly 1 in total
    const float lse = log1pf((float)(total - 1)), lse1 = TWO ? log1pf((float)(total1 - 1)) : lse;
    double kd = 0, P = 0, rest = 0;
    // the rest: the classes that the teacher does not list, relative to their maximum
    const float top_rest = extra ? fmaxf(a.m, x_y) : a.m;
    const float down = exp2_fast((a.m - top_rest) * c);
    o.y_rest = extra ? exp2_fast((x_y - top_rest) * c) : 0.f;
    const float sum_rest = a.s * down + o.y_rest;
    o.scale = 1.f;
    if (k > 0 && tail) {
        P = p;
        kd = l + lse * p;
        if (sum_rest != 0.f) {
            rest = p > 1 ? 0 : 1 - p;
            if (rest != 0)
                kd += rest * (logf((float)rest) -
                              (logf(sum_rest) + ((double)top_rest - ref) * inv_td - lse));
            P += rest;
        }
    } else if (k > 0 && p != 0) {
        const double to_one = 1 / p;
        o.scale = (float)to_one;
        P = p * to_one;  // 1, or NaN
        kd = l * to_one - logf((float)p) + lse;
    } else if (k > 0) {
        kd = 0.f * lse;  // entries without probability: 0, or NaN
    }
    const float per_rest = rest == 0 ? 0.f : (float)rest / sum_rest;
    o.y_rest *= per_rest;
    double v = k > 0 ? (double)t.soft * temperature * temperature * kd : 0;
    if (label) v += (double)t.hard * ((double)lse1 - ((double)x_y - ref));
    o.loss = o.empty || o.none ? 0.f : (float)(w * v);
    o.soft = k > 0 ? -w * t.soft * temperature : 0.f;
    o.hard = label ? -w * t.hard : 0.f;
    o.P_total = o.empty ? 0.f : (float)P / (float)total;
    o.one_total = o.empty ? 0.f : 1.f / (float)total1;
    o.K = o.soft == 0.f ? 0.f : o.soft * (o.P_total * up - per_rest * down);
    o.K1 = o.hard == 0.f ? 0.f : o.hard * o.one_total * up1;
    if (!TWO) o.K += o.K1;
    return o;
}

// What a launch does: all of it, a row to a workgroup; or, for rows in parts,
// first the statistics of the dense classes, a workgroup each part, and the
// listed classes, one workgroup more; then the delta.
enum { WHOLE, STATS, DELTA };

// What the first of two launches leaves for the second.
struct RowList {
    Listed listed[LISTED_WAVES];
    float x_y;
    int extra;
    Entry entry[ACH_TOP_MAX + 1];
};
struct Between {
    RowList *list;
    Dense *dense;
};

// The losses of rows in parts, and their sum: a workgroup of its own in the
// second launch, a row to a thread.
template <int TWO, int NT>
__device__ __forceinline__ void part_losses(const ach_logits_desc &d, const ach_distill_desc &t,
                                            const int32_t *labels, const float *row_weights,
                                            float *loss, float *cost, int parts,
                                            const Between &between)
{
    __shared__ double sums[NT / 64];
    const int k = t.soft != 0.f ? t.k : 0, r = threadIdx.x;
    const float c = LOG2E / d.temperature;
    const float w = r >= d.rows ? 0.f : row_weights ? row_weights[r] : 1.f;
    float v = 0.f;
    if (w != 0.f) {
        Dense a = {-FLT_MAX, 0.f, 0.f};
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
            Dense o = between.dense[(size_t)r * parts + i];
            const float m = fmaxf(a.m, o.m);
            raise_dense<BOTH>(a, m, c);
            raise_dense<BOTH>(o, m, c);
            a.s += o.s;
            a.s1 += o.s1;
        }
        const int y = t.hard != 0.f ? labels[r] : -1;
        const RowList &list = between.list[r];
        v = row_terms<TWO>(a, list.listed, min(NT / 64, (k >> 6) + 1), t, k, d.temperature,
                           y >= 0 && y < d.classes, list.extra, list.x_y, w)
                .loss;
    }
    if (loss && r < d.rows) loss[r] = v;
    if (!cost) return;
    const double sum = block_sum<NT>((double)v, sums);
    if (r == 0) *cost = (float)sum;
}

// 2048 x 131072 bf16, 64 entries: 266 us, 4.0 TB/s of logits read once and the
// delta; the second reading comes from HBM in part, as the rows in flight, four a
// compute unit, fill the 256 MB cache.  Fewer leave the waits of a row's start
// and middle open (three: 312 us, two: 346).
template <int TYPE, int NT, int TWO, int MODE>
__global__ void __launch_bounds__(NT, 4)
    k_distill(ach_logits_desc d, ach_distill_desc t, const typename Elem<TYPE>::T *logits,
              const int32_t *__restrict__ teacher_ids, const void *__restrict__ teacher_values,
              const int32_t *__restrict__ labels, const float *__restrict__ row_weights,
              float *loss, typename Elem<TYPE>::T *delta, int64_t delta_stride, float *row_loss,
              int parts, int span, int stashed, Between between, bool past, float *cost)
{
    using T = typename Elem<TYPE>::T;
    typedef typename Row<TYPE>::Chunk Chunk;
    constexpr int V = Row<TYPE>::VEC, W = NT / 64;
    __shared__ DistillLds<NT> sh;
    const int k = t.soft != 0.f ? t.k : 0;
    const bool tail = t.mode == ACH_DISTILL_TAIL;
    const float c = LOG2E / d.temperature;
    const double inv_td = 1. / d.temperature;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int groups = MODE == STATS ? parts + 1 : parts;
    if (MODE == DELTA && blockIdx.x == (unsigned)(d.rows * parts)) {
        part_losses<TWO, NT>(d, t, labels, row_weights, loss, cost, parts, between);
        return;
    }
    for (size_t b = blockIdx.x; b < (size_t)d.rows * groups; b += gridDim.x) {
        const int r = (int)(b / groups), part = (int)(b % groups), at = part * span;
        const T *row = logits + (size_t)r * d.stride;
        const Range<TYPE> g = {row + at, at, min(span, d.classes - at)};
        const float w = row_weights ? row_weights[r] : 1.f;
        if (w == 0.f) {
            if (MODE != STATS && delta) {
                T *out = delta + (size_t)r * delta_stride + at;
                const Chunk zero = {};
                for (int q = threadIdx.x; q < g.chunks(); q += NT)
                    Row<TYPE>::template store<false>(out + (size_t)q * V, zero);
                if (threadIdx.x < g.rest()) out[g.chunks() * V + threadIdx.x] = (T)0.f;
            }
            if (MODE == WHOLE && threadIdx.x == 0) {
                if (loss) loss[r] = 0.f;
                if (row_loss) row_loss[r] = 0.f;
            }
            continue;
        }
        int y = t.hard != 0.f ? labels[r] : -1;
        if (y < 0 || y >= d.classes) y = -1;
        RowList *list = MODE == WHOLE ? nullptr : between.list + r;
        const int waves = min(W, (k >> 6) + 1);  // that have listed classes
        Entry entry;
        Dense a = {-FLT_MAX, 0.f, 0.f};
        if (MODE != DELTA) {
            __syncthreads();  // of the last row
            for (int i = threadIdx.x; i <= k; i += NT) {
                const int id = i < k ? teacher_ids[(size_t)r * k + i] : y;
                sh.id[i] = id < 0 || id >= d.classes ? -1 : id;
                sh.repeated[i] = 0;
            }
            if (threadIdx.x == 0) sh.x_y = 0.f;
        }
        if (MODE == WHOLE || (MODE == STATS && part == parts)) {
            __syncthreads();
            find_repeated<NT>(k, sh);
            __syncthreads();
            if (threadIdx.x == 0) sh.extra = y >= 0 && !sh.repeated[k];
            listed_terms<TYPE, NT, TWO>(entry, row, teacher_values, t.teacher_type,
                                        (size_t)r * k, k, tail, d.temperature, inv_td, sh);
        }
        if (MODE == STATS && part == parts) {
            __syncthreads();
            if ((int)threadIdx.x < waves) list->listed[threadIdx.x] = sh.listed[threadIdx.x];
            if (threadIdx.x == 0) {
                list->x_y = sh.x_y;
                list->extra = sh.extra;
            }
            if ((int)threadIdx.x <= k) list->entry[threadIdx.x] = entry;
            continue;
        }
        if (MODE == DELTA) {
            if (lane < parts) a = between.dense[(size_t)r * parts + lane];
            wave_dense<BOTH>(a, c);
        } else {
            a = stream_dense<TYPE, NT, TWO>(g, c, k, stashed, sh);
            wave_dense<TWO>(a, c);
            if (!TWO) a.s1 = a.s;
            if (lane == 0) sh.wave[wave] = a;
            __syncthreads();
            a = sh.wave[0];
#pragma unroll 1
            for (int i = 1; i < W; ++i) {
                Dense o = sh.wave[i];
                const float m = fmaxf(a.m, o.m);
                raise_dense<TWO>(a, m, c);
                raise_dense<TWO>(o, m, c);
                a.s += o.s;
                a.s1 = TWO ? a.s1 + o.s1 : a.s;
            }
        }
        if (MODE == STATS) {
            if (threadIdx.x == 0) between.dense[(size_t)r * parts + part] = a;
            continue;
        }
        const RowTerms terms =
            row_terms<TWO>(a, MODE == DELTA ? list->listed : sh.listed, waves, t, k, d.temperature,
                           y >= 0, MODE == DELTA ? list->extra : sh.extra,
                           MODE == DELTA ? list->x_y : sh.x_y, w);
        if (MODE == WHOLE && threadIdx.x == 0) {
            if (loss) loss[r] = terms.loss;
            if (row_loss) row_loss[r] = terms.loss;
        }
        if (!delta) continue;
        T *out = delta + (size_t)r * delta_stride + at;
        if (terms.none) {  // a short loop: a second copy of the one above costs others 2%
#pragma unroll 1
            for (int j = threadIdx.x; j < g.len; j += NT) out[j] = (T)0.f;
            continue;
        }
        const auto grad = [&](float v) {
            const float x = v - terms.m, e = exp2_fast(x * c);
            float o = terms.K * e;
            if (TWO) o = fmaf(terms.K1, second<TWO>(e, x), o);
            return (T)o;
        };
        const int n = g.chunks();
        extern __shared__ uint4 stash[];
        const int stash_chunks = MODE == WHOLE ? stashed * UNROLL * NT : 0;
        const auto write = [&](auto PAST) {
            // from the end, which the caches hold
            constexpr int U = UNROLL;
            for (int q = n - 1 - (int)threadIdx.x; q >= 0; q -= U * NT) {
                Chunk v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (q - u * NT >= stash_chunks)
                        v[u] = Row<TYPE>::load(g.p + (size_t)(q - u * NT) * V);
                    else if (q - u * NT >= 0)
                        __builtin_memcpy(&v[u], &stash[q - u * NT], 16);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (q - u * NT < 0) break;
                    Chunk o;
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = grad((float)v[u][i]);
                    Row<TYPE>::template store<PAST.value>(out + (size_t)(q - u * NT) * V, o);
                }
            }
        };
        if (past) write(Flag<true>());
        else write(Flag<false>());
        if (threadIdx.x < g.rest()) {
            const int j = n * V + threadIdx.x;
            out[j] = grad((float)g.p[j]);
        }
        __syncthreads();  // the listed classes over what was written for them
        const int i = threadIdx.x, of = i >> 6;
        if (MODE == DELTA && i <= k) entry = list->entry[i];
        if (i <= k && entry.id >= at && entry.id < at + g.len) {
            const auto own = [&](const float (&to)[LISTED_WAVES]) {
                return of == 0 ? to[0] : of == 1 ? to[1] : to[2];
            };
            const float e = entry.e * own(terms.to_e), e1 = entry.e1 * own(terms.to_e1),
                        p = entry.p * own(terms.to_p) * terms.scale;
            float v = 0.f;
            if (terms.soft != 0.f)
                v = terms.soft * (terms.P_total * e - (i < k ? p : terms.y_rest));
            if (terms.hard != 0.f)
                v += terms.hard * (terms.one_total * e1 - (entry.id == y ? 1.f : 0.f));
            out[entry.id - at] = (T)(terms.empty ? 0.f : v);
        }
    }
}

// The sum of the rows' losses in a fixed order, eight loads in flight a thread
// (one after the other, 4096 of them took 256 threads longer than their rows).
constexpr int SUM_THREADS = 1024;
__global__ void __launch_bounds__(SUM_THREADS) k_sum_losses(const float *__restrict__ row_loss,
                                                            int rows, float *cost)
{
    constexpr int U = 8;
    __shared__ double sh[SUM_THREADS / 64];
    double s = 0;
    for (size_t first = threadIdx.x; first < (size_t)rows; first += U * SUM_THREADS) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t i = first + u * SUM_THREADS;
            v[u] = i < (size_t)rows ? row_loss[i] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) s += v[u];
    }
    s = block_sum<SUM_THREADS>(s, sh);
    if (threadIdx.x == 0) *cost = (float)s;
}

// ---- plans ---------------------------------------------------------------------------
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
// (at most 256) and long.
struct Split {
    int parts, span;
};

Split split_rows(int rows, int classes, int least)
{
    int parts = rows > 0 ? 512 / rows : 1;  // two workgroups a compute unit
    parts = parts < classes / 4096 ? parts : classes / 4096;
    if (parts > MOST_PARTS) parts = MOST_PARTS;
    if (parts < 2 || classes < least) return {1, classes};
    const int span = (int)((((int64_t)classes + parts - 1) / parts + 63) / 64 * 64);
    return {(int)(((int64_t)classes + span - 1) / span), span};
}

// The second launch is worth its time from about 64 K classes in the forward
// pass (1 row, bf16, 20 alternatives: 32768 classes 9.3 us in one launch, 11.5
// in two; 100003 classes, 64 rows: 21 and 15.6), and from 16 K in distillation,
// whose two passes over a row are both shared out (16 rows of 32768: 16.0 and
// 11.7 us).
constexpr int SPLIT_LOGPROBS = 65536, SPLIT_DISTILL = 16384;

// Threads of a workgroup of the forward pass.  A wave by itself needs no
// barriers, which pays for short rows, or up to 8192 classes where there are
// enough rows to fill the chip with single waves (2048 x 8192 bf16: 15.3 us, 21.8 with
// 256 threads); the bound on the k-th largest wants k of its lanes.  Few long
// rows take 512 (512 x 65536 fp32: 33 us, 40 with 256); more rows 256 (4096 x
// 32768 bf16: 55 us, 120 with 1024).
int threads_logprobs(int rows, const Split &s, int k)
{
    if (s.span <= (rows >= 1024 ? 8192 : 2048) && k <= 32) return 64;
    return (int64_t)rows * s.parts < 1024 && s.span >= 16384 ? 512 : 256;
}

// The same of distillation; the listed classes have a thread each.
int threads_distill(int rows, const Split &s, int k)
{
    if (s.parts > 1) return 256;
    if (s.span <= 2048 && k < 64) return 64;
    return rows < 256 && s.span >= 8192 ? 512 : 256;
}

// Gradients of more than the L2 caches hold (8 of 4 MB) are stored past them:
// what reads them next finds them in memory either way, and the logits that
// the kernel reads a second time stay cached.
bool past_caches(const ach_logits_desc &d)
{
    return (size_t)d.rows * d.classes * elem_size(d.type) > (size_t)32 << 20;
}

unsigned grid_of(size_t n) { return (unsigned)(n < (1u << 20) ? n : 1u << 20); }

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_logprobs_workspace(const ach_logits_desc *desc, int k)
{
    ach_logits_desc d;
    if (!logits_desc(desc, &d) || k < 0 || k > ACH_TOP_MAX || k > d.classes) return 0;
    const Split s = split_rows(d.rows, d.classes, SPLIT_LOGPROBS);
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
    const Split sp = split_rows(d.rows, d.classes, SPLIT_LOGPROBS);
    const int nt = threads_logprobs(d.rows, sp, k);
    const dim3 grid(grid_of((size_t)d.rows * sp.parts));
    Total *part = (Total *)ws;
    uint64_t *lists = (uint64_t *)(part + (size_t)d.rows * sp.parts);
    const LogprobsOut o = {logprobs, ranks, entropy, stats, top_ids, top_logprobs};
    hipStream_t st = as_stream(s);
#define GO(TYPE, NT, FULL, TOP)                                                                   \
    hipLaunchKernelGGL((k_logprobs<TYPE, NT, FULL, TOP>), grid, dim3(NT), 0, st, d,               \
                       (const Elem<TYPE>::T *)logits, ids, k, o, sp.parts, sp.span, part, lists)
#define WITH(TYPE, FULL, TOP)                                                                     \
    do {                                                                                          \
        if (nt == 64) GO(TYPE, 64, FULL, TOP);                                                    \
        else if (nt == 512) GO(TYPE, 512, FULL, TOP);                                             \
        else GO(TYPE, 256, FULL, TOP);                                                            \
    } while (0)
#define CALL(TYPE)                                                                                \
    do {                                                                                          \
        if (entropy || ranks) {                                                                   \
            if (k) WITH(TYPE, true, true);                                                        \
            else WITH(TYPE, true, false);                                                         \
        } else if (k) WITH(TYPE, false, true);                                                    \
        else WITH(TYPE, false, false);                                                            \
    } while (0)
    FOR_TYPE(d.type, CALL);
#undef CALL
#undef WITH
#undef GO
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
    const bool past = past_caches(d);
    hipStream_t st = as_stream(s);
#define CALL(TYPE)                                                                                \
    hipLaunchKernelGGL((k_logprobs_bwd<TYPE>), grid, block, 0, st, d,                             \
                       (const Elem<TYPE>::T *)logits, ids, stats, entropy, dlogprobs, dentropy,   \
                       (Elem<TYPE>::T *)dlogits, dstride, parts, span, past)
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
    const Split s = split_rows(d.rows, d.classes, SPLIT_DISTILL);
    size_t n = round16((size_t)d.rows * sizeof(float));
    if (s.parts > 1)
        n += (size_t)d.rows * (sizeof(RowList) + s.parts * sizeof(Dense));
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
        const Split sp = split_rows(d.rows, d.classes, SPLIT_DISTILL);
        const int two = t.soft == 0.f || t.hard == 0.f || d.temperature == 1.f ? ONE
                        : d.temperature == 2.f                                 ? SQUARE
                        : d.temperature == 4.f                                 ? FOURTH
                                                                               : BOTH;
        if (t.soft == 0.f) d.temperature = 1.f;  // the label's term is at temperature 1
        const dim3 grid(grid_of((size_t)d.rows * sp.parts));
        const int nt = threads_distill(d.rows, sp, t.soft != 0.f ? t.k : 0);
        const bool past = past_caches(d);
        float *row_loss = (float *)ws;
        RowList *list = (RowList *)((char *)ws + round16((size_t)d.rows * sizeof(float)));
        const Between between = {list, (Dense *)(list + d.rows)};
        // few rows (split_rows): a workgroup each, and one for the losses
        const dim3 stats_grid(d.rows * (sp.parts + 1)), delta_grid(d.rows * sp.parts + 1);
        // Of a row that a workgroup reads twice, the first turns stay in LDS in
        // between, 32 KB (four workgroups a compute unit still fit).  With 64
        // entries, without and with: 4096 x 32768 bf16 140 and 129 us, 2048 x
        // 131072 273 and 266; 1021 x 50021 fp16 with 17 entries 64.0 and 61.1.
        const int turn_bytes = UNROLL * nt * 16;
        int stashed = (int)((size_t)d.classes * elem_size(d.type) / turn_bytes);
        const int room = sp.parts > 1 || !delta ? 0 : 32768 / turn_bytes;
        stashed = stashed < room ? stashed : room;
        const size_t lds = (size_t)stashed * turn_bytes;
#define GO(TYPE, NT, TWO, MODE, GRID)                                                             \
    hipLaunchKernelGGL((k_distill<TYPE, NT, TWO, MODE>), GRID, dim3(NT), lds, st, d, t,           \
                       (const Elem<TYPE>::T *)logits, teacher_ids, teacher_values, labels,        \
                       row_weights, loss, (Elem<TYPE>::T *)delta, delta_stride, row_loss,         \
                       sp.parts, sp.span, stashed, between, past, cost)
#define WITH(TYPE, TWO)                                                                           \
    do {                                                                                          \
        if (sp.parts > 1) {                                                                       \
            GO(TYPE, 256, TWO, STATS, stats_grid);                                                \
            GO(TYPE, 256, TWO, DELTA, delta_grid);                                                \
        } else if (nt == 64) GO(TYPE, 64, TWO, WHOLE, grid);                                      \
        else if (nt == 512) GO(TYPE, 512, TWO, WHOLE, grid);                                      \
        else GO(TYPE, 256, TWO, WHOLE, grid);                                                     \
    } while (0)
#define CALL(TYPE)                                                                                \
    do {                                                                                          \
        if (two == ONE) WITH(TYPE, ONE);                                                          \
        else if (two == SQUARE) WITH(TYPE, SQUARE);                                               \
        else if (two == FOURTH) WITH(TYPE, FOURTH);                                               \
        else WITH(TYPE, BOTH);                                                                    \
    } while (0)
        FOR_TYPE(d.type, CALL);
#undef CALL
#undef WITH
#undef GO
        const int rc = check_launch();
        if (rc || !cost || sp.parts > 1) return rc;
    }
    if (!cost) return ACH_OK;
    hipLaunchKernelGGL(k_sum_losses, dim3(1), dim3(SUM_THREADS), 0, st, (const float *)ws, d.rows,
                       cost);
    return check_launch();
}

}  // extern "C"
