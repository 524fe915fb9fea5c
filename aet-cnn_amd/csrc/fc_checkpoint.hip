// A fully connected layer's weight gradient from its input's 8-bit checkpoint
// (include/aetcnn_ops.h): dw = delta^T x on the bf16 matrix instructions.
//
// A code times its power of two is a bf16 number, and so is each piece of a
// delta (its first 8 bits, the next 8, the last 8; one piece for bf16, two for
// fp16, three for fp32): every product is exact and is summed in fp32.  The last two
// pieces of fp32 are scaled by kPieceUp, as those of values under 2^-110 would lie below
// bf16's smallest number (a relative error of 1e-6 at 2^-115, 1e-4 at 2^-122).  Sums that
// are not finite so, near deltas or sums of 2^111, are done again in fp32.  (Scaling and
// that check: 128 x 9216 -> 4096 47.7 us, without 47.0, 256 rows 74 and 71.)
//
// Tiles of 256 outputs x 128 inputs or 128 x 256, on few rows 128 x 128, a wave 64 x
// 64 (bf16 also 128 x 64) of it.  A stage of 32 rows of both operands is loaded two
// stages ahead, turned into bf16 and stored as it lies in memory, [row][column]; the
// matrix instructions want 8 rows of a column in a lane, which the transposing LDS
// loads give: 16 lanes read 4 rows x 16 columns, and each gets a column of it.  Few
// tiles share out the rows in slices, whose sums a second launch adds up in order.
//
// Bound by the matrix units on many rows: 8192 x 8192 -> 4096 bf16 503 us, 1090
// TFLOP/s (a matrix product of the library at 8192^3 in bf16: 1250); fp32 1340 us,
// three passes of 415; 16384 x 4096 -> 1024 bf16 151 us, of which 14 are the four
// slices' sums.  On few rows by the writing of dw, which two workgroups a compute unit
// overlap in part with a tile's start and its stages: 128 x 9216 -> 4096 fp32 47 us for
// 154 MB, fp16 37, bf16 31.  What it took on 16384 x 4096 -> 1024 bf16: one stage ahead
// 399 us, two 233; offsets in the loads' windows instead of 64-bit addresses and clamps
// (100 vector instructions for 8 of the matrix) 189; waves of 128 x 64 162; the
// operands' loads among the matrix instructions 155; a last turn that loads nothing
// 153.  Several tiles a workgroup, the next one's loads before the writing, lost 10% on
// many rows, where it spoils the loop's order.
#include "checkpoint.hpp"
#include "pieces.hpp"

#include <math.h>

namespace ach {
namespace {

constexpr int DEPTH = 32;  // rows of a stage
constexpr int RING = 2;    // stages in flight (the loops are written for two)
constexpr int MOST_SLICES = 64;
constexpr int MOST_COLUMNS = 1 << 23;  // inputs, outputs, stride: a stage's offsets fit 31 bits

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

template <int TYPE> struct Pieces {
    static constexpr int N = TYPE == ACH_F32 ? 3 : TYPE == ACH_F16 ? 2 : 1;
};

struct Fc {
    int rows, inputs, outputs;
    int64_t stride;
    Kept k;
    float *dw, *part;  // part: [slices][outputs][inputs], or null
    int accumulate;
    int span;          // rows of a slice
    int ti;            // tiles along the inputs
    bool past;         // dw past the caches
};

// The upper halves of two floats: their first 8 bits of precision as bf16.
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi)
{
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
}
__device__ __forceinline__ float below(float x)  // what they leave
{
    return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}

// Eight values of a delta, and the pieces whose sum they are.
template <int TYPE> struct Eight {
    static constexpr int N = TYPE == ACH_F32 ? 2 : 1;  // loads of 16 bytes
    v4u w[N];
    // moves 16-bit value i + by to value i, for a chunk that was loaded `by` early
    __device__ __forceinline__ void shift(int by)
    {
        v4u u = w[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = by & 4 ? u[(i + 2) & 3] : u[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = by & 2 ? u[(i + 1) & 3] : u[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = by & 1 ? u[i] >> 16 | u[(i + 1) & 3] << 16 : u[i];
        w[0] = u;
    }
    __device__ __forceinline__ void split(v4u *p) const
    {
        if constexpr (TYPE == ACH_BF16) {
            p[0] = w[0];
        } else {
            float f[8];
            if constexpr (TYPE == ACH_F32) {
                __builtin_memcpy(f, w, sizeof(f));
            } else {
                _Float16 h[8];
                __builtin_memcpy(h, w, sizeof(h));
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float a = f[2 * i], b = f[2 * i + 1];
#pragma unroll
                for (int q = 0; q < Pieces<TYPE>::N; ++q) {
                    p[q][i] = upper_halves(a, b);
                    a = below(a), b = below(b);
                    if (TYPE == ACH_F32 && q == 0) a *= kPieceUp, b *= kPieceUp;
                }
            }
        }
    }
};

// A window of DEPTH rows on a matrix, moved from stage to stage; what lies behind
// the last byte reads as 0.
struct Window {
    const char *p;
    int64_t left, step;
    __device__ __forceinline__ Window(const void *base, int64_t pitch, int64_t row_bytes, int r, int end)
        : p((const char *)base + r * pitch), left((end - r) * pitch - (pitch - row_bytes)),
          step(DEPTH * pitch)
    {
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t next()
    {
        const __amdgpu_buffer_rsrc_t w =
            make_rsrc(p, (unsigned)max(min(left, (int64_t)0x7fffffff), (int64_t)0));
        p += step, left -= step;
        return w;
    }
};

// Eight columns' rows of a tile in LDS as a lane's operand of a 16-row step: `p`
// is the lane's own place in the first four rows.
template <int PITCH> __device__ __forceinline__ v8bf fragment(const short *p)
{
    typedef __attribute__((address_space(3))) v4s *Lds;
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p),
              b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * PITCH));
    const v8s v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(v8bf, v);
}

// How a chunk of delta is loaded.  What lies behind the last output or input is
// never stored, so any values will do there: loads that pass a row's end read the
// next row, or zeros behind the last one (WHOLE).  The range check is by dwords, so
// 16-bit values, which would lose the last one of an odd number, are loaded whole
// chunks inside a row instead, early and then shifted (EARLY), or one by one
// (SINGLE, under 8 outputs; its 16 loads a stage take addresses that in fp16 tiles of 128 x
// 128 lie in part in memory, six of them read back in the loop: 1000 x 3000 -> 6 11.5 us).
enum { WHOLE, EARLY, SINGLE };

// The sums of a lane's outputs o .. o + 3, o + 8 .. in fp32, for inputs i and i + 32.
template <int TYPE>
__device__ __forceinline__ void plain_sums(const typename Elem<TYPE>::T *delta, const Fc &a, int r0, int r1,
                                           int o, int i, float (*v)[16])
{
    // (what lies behind the last output or input is not written)
    const int first = min(i, a.k.width - 1), second = min(i + 32, a.k.width - 1);
#pragma unroll
    for (int e = 0; e < 16; ++e) v[0][e] = v[1][e] = 0.f;
    for (int r = r0; r < r1; ++r) {
        const int8_t *const codes = a.k.codes + (size_t)r * a.k.width;
        const uint8_t *const steps = a.k.steps + (size_t)r * (a.k.width / KEPT_BLOCK);
        const float x0 = (float)codes[first] * kept_scale(steps[first / KEPT_BLOCK]),
                    x1 = (float)codes[second] * kept_scale(steps[second / KEPT_BLOCK]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float d = (float)delta[r * a.stride + min(o + 8 * (e >> 2) + (e & 3), a.outputs - 1)];
            v[0][e] = fmaf(d, x0, v[0][e]);
            v[1][e] = fmaf(d, x1, v[1][e]);
        }
    }
}

// WO x WI waves of 32 MO outputs x 64 inputs
template <int TYPE, int WO, int WI, int MO> struct Tile {
    static constexpr int THREADS = 64 * WO * WI;
    static constexpr int O = 32 * MO * WO, I = 64 * WI;
    static constexpr int OP = O + 32, IP = I + 32;  // 16-bit values of an LDS row
    struct Stage {
        short d[Pieces<TYPE>::N][DEPTH * OP], x[DEPTH * IP];
    };
    static constexpr int TP = I + 4;  // floats of a row of the tile on its way out
    static constexpr size_t OUT = 32 * WO * TP * sizeof(float);
    static constexpr size_t LDS = 2 * sizeof(Stage) > OUT ? 2 * sizeof(Stage) : OUT;
};

// (fp32 tiles of 128 x 256 keep three values for after the loop in memory.)
template <int TYPE, int WO, int WI, int MO, int HOW>
__global__ void __launch_bounds__(64 * WO * WI, 2)
k_fc_wgrad(const typename Elem<TYPE>::T *delta, Fc a)
{
    using S = Tile<TYPE, WO, WI, MO>;
    constexpr int P = Pieces<TYPE>::N, SIZE = sizeof(typename Elem<TYPE>::T);
    constexpr int XC = DEPTH * S::I / S::THREADS;        // codes of a thread's load: 8 or 16
    constexpr int DN = DEPTH * S::O / S::THREADS / 8;    // chunks of 8 values of delta
    constexpr int DR = S::THREADS / (S::O / 8);          // rows apart
    extern __shared__ __align__(16) char smem[];
    typename S::Stage *const stage = reinterpret_cast<typename S::Stage *>(smem);
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wo = wave % WO, wi = wave / WO;
    // each XCD, which takes every eighth workgroup, gets a contiguous range of
    // tiles, which share their operands in its L2
    const int xcd = blockIdx.x & 7, tiles = gridDim.x;
    const int tile = xcd * (tiles >> 3) + min(xcd, tiles & 7) + (int)(blockIdx.x >> 3);
    const int o0 = tile / a.ti * S::O, i0 = tile % a.ti * S::I;
    const int r0 = (int)blockIdx.y * a.span, r1 = min((int64_t)a.rows, (int64_t)r0 + a.span);

    // a thread's share of a stage
    const int xr = tid / (S::I / XC), xc = tid % (S::I / XC) * XC;
    const int dr = tid / (S::O / 8), dc = tid % (S::O / 8) * 8;
    const int64_t pitch = a.stride * SIZE;
    struct Load {
        uint32_t codes[XC / 4], step;
        Eight<TYPE> d[DN];
    };
    const int x_col = min(i0 + xc, a.k.width - XC);
    const int x_at = xr * a.k.width + x_col, s_at = x_at / KEPT_BLOCK;
    const int d_col = HOW == EARLY ? min(o0 + dc, a.outputs - 8) : o0 + dc;
    const int late = min(o0 + dc - d_col, 7);
    int d_at[DN];
#pragma unroll
    for (int h = 0; h < DN; ++h) d_at[h] = (dr + h * DR) * (int)pitch + d_col * SIZE;
    Window codes(a.k.codes, a.k.width, a.k.width, r0, r1),
        steps(a.k.steps, a.k.width / KEPT_BLOCK, a.k.width / KEPT_BLOCK, r0, r1),
        deltas(delta, pitch, (int64_t)a.outputs * SIZE, r0, r1);
    auto load = [&](Load &g) {
        const __amdgpu_buffer_rsrc_t c = codes.next(), t = steps.next(), d = deltas.next();
        if constexpr (XC == 16) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(c, x_at, 0, 0);
            __builtin_memcpy(g.codes, &v, 16);
        } else {
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(c, x_at, 0, 0);
            __builtin_memcpy(g.codes, &v, 8);
        }
        g.step = __builtin_amdgcn_raw_buffer_load_b8(t, s_at, 0, 0);
#pragma unroll
        for (int h = 0; h < DN; ++h) {
            if constexpr (HOW == SINGLE) {
                uint16_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = __builtin_amdgcn_raw_buffer_load_b16(d, d_at[h] + 2 * i, 0, 0);
                __builtin_memcpy(g.d[h].w, v, sizeof(v));
            } else {
#pragma unroll
                for (int i = 0; i < Eight<TYPE>::N; ++i) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b128(d, d_at[h] + 16 * i, 0, 0);
                    __builtin_memcpy(&g.d[h].w[i], &v, 16);
                }
            }
        }
    };
    auto store = [&](Load &g, int s) {
        const float scale = kept_scale(g.step);
        uint32_t w[XC / 2];
#pragma unroll
        for (int i = 0; i < XC / 4; ++i) {
            float f[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) f[b] = (float)(int8_t)(g.codes[i] >> (8 * b)) * scale;
            w[2 * i] = upper_halves(f[0], f[1]);
            w[2 * i + 1] = upper_halves(f[2], f[3]);
        }
        short *const to = &stage[s].x[xr * S::IP + xc];
#pragma unroll
        for (int i = 0; i < XC / 8; ++i) *(v4u *)(to + 8 * i) = *(v4u *)(w + 4 * i);
#pragma unroll
        for (int h = 0; h < DN; ++h) {
            v4u p[P];
            if constexpr (HOW == EARLY) g.d[h].shift(late);
            g.d[h].split(p);
#pragma unroll
            for (int q = 0; q < P; ++q) *(v4u *)&stage[s].d[q][(dr + h * DR) * S::OP + dc] = p[q];
        }
    };
    v16f hi[MO][2], lo[P > 1 ? MO : 1][2];
#pragma unroll
    for (int i = 0; i < MO; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) hi[i][j][e] = lo[P > 1 ? i : 0][j][e] = 0.f;

    // a lane's place in a 16-row step: row 8 * (lane / 32) + lane % 16 / 4, column
    // 16 * (lane / 16 % 2) + 4 * (lane % 4)
    const int row = 8 * (lane >> 5) + ((lane & 15) >> 2), column = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    const int d_place = row * S::OP + wo * 32 * MO + column, x_place = row * S::IP + wi * 64 + column;
    auto multiply = [&](int s) {
        __builtin_amdgcn_iglp_opt(0);  // operand loads among the matrix instructions
#pragma unroll
        for (int step = 0; step < DEPTH; step += 16) {
            v8bf x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) x[j] = fragment<S::IP>(&stage[s].x[x_place + step * S::IP + j * 32]);
#pragma unroll
            for (int i = 0; i < MO; ++i) {
                v8bf p[P];
#pragma unroll
                for (int q = 0; q < P; ++q)
                    p[q] = fragment<S::OP>(&stage[s].d[q][d_place + step * S::OP + i * 32]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    hi[i][j] = MFMA_BF(p[0], x[j], hi[i][j]);
#pragma unroll
                    for (int q = 1; q < P; ++q) lo[i][j] = MFMA_BF(p[q], x[j], lo[i][j]);
                }
            }
        }
    };
    Load ring[RING];
#pragma unroll
    for (int u = 0; u < RING; ++u) load(ring[u]);
    store(ring[0], 0);
    load(ring[0]);
    __syncthreads();
    for (int r = r0; r + RING * DEPTH < r1; r += RING * DEPTH) {
#pragma unroll
        for (int u = 1; u <= RING; ++u) {
            multiply((u + 1) % 2);
            store(ring[u % RING], u % 2);
            load(ring[u % RING]);
            __syncthreads();
        }
    }
    multiply(0);  // the last turn, with nothing left to load (a stage behind the last row is zeros)
    store(ring[1], 1);
    __syncthreads();
    multiply(1);
    if constexpr (TYPE == ACH_F32) {
        // (an infinite delta leaves NaN of the other pieces)
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < MO; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) all = __builtin_elementwise_maximum(all, fabsf(lo[i][j][e]));
        if (__builtin_expect(__any(!(all < INFINITY)), 0)) {
#pragma unroll
            for (int i = 0; i < MO; ++i) {
                float v[2][16];
                plain_sums<TYPE>(delta, a, r0, r1, o0 + (wo * MO + i) * 32 + 4 * (lane >> 5),
                                 i0 + wi * 64 + (lane & 31), v);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!(fabsf(lo[i][j][e]) < INFINITY)) hi[i][j][e] = v[j][e], lo[i][j][e] = 0.f;
            }
        }
    }

    float *const out = a.part ? a.part + (size_t)blockIdx.y * a.outputs * a.inputs : a.dw;
    const bool add = a.accumulate && !a.part;
    // 32 outputs of each wave at a time through LDS, so that a row of the tile is written by
    // consecutive lanes, 16 bytes each (128 x 9216 -> 4096 fp32 51 us, bf16 34; from the
    // registers, 128 bytes of two rows a time, 56 and 43)
    float *const turned = reinterpret_cast<float *>(smem);
    constexpr int CHUNKS = S::I / 4, ROWS = S::THREADS / CHUNKS;
    const int col = i0 + tid % CHUNKS * 4, left = a.inputs - col;
#pragma unroll
    for (int i = 0; i < MO; ++i) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                turned[(wo * 32 + 4 * (lane >> 5) + 8 * (e >> 2) + (e & 3)) * S::TP + wi * 64 + j * 32 +
                       (lane & 31)] = TYPE == ACH_F32 ? fmaf(lo[P > 1 ? i : 0][j][e], 1 / kPieceUp, hi[i][j][e])
                                      : P > 1         ? hi[i][j][e] + lo[P > 1 ? i : 0][j][e]
                                                      : hi[i][j][e];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 32 * WO / ROWS; ++k) {
            const int r = tid / CHUNKS + k * ROWS, o = o0 + ((r >> 5) * MO + i) * 32 + (r & 31);
            if (o >= a.outputs) continue;
            float *const p = out + (size_t)o * a.inputs + col;
            float v[4];
            __builtin_memcpy(v, __builtin_assume_aligned(&turned[r * S::TP + tid % CHUNKS * 4], 16), 16);
            if (add) {
                float w[4];
                load_floats<4>(p, 0, left, 0.f, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += w[e];
            }
            if (a.past) store_values<ACH_F32, true>(p, left, v);
            else store_values<ACH_F32>(p, left, v);
        }
    }
}

// dw (+)= the slices' sums, four values and eight slices in flight a thread (20000 x
// 30 -> 20 fp32, 64 slices: 24.0 us with four, 21.6 with eight).
__global__ void __launch_bounds__(256)
k_fc_wgrad_join(const float *part, size_t n, int slices, float *dw, int accumulate)
{
    constexpr int U = 8;
    for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (size_t)gridDim.x * 1024) {
        const int left = (int)(n - i < 4 ? n - i : 4);
        float s[4], v[U][4];
        load_floats<4>(accumulate ? dw : nullptr, i, left, 0.f, s);
        for (int k = 0; k < slices; k += U) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                load_floats<4>(k + u < slices ? part : nullptr, (size_t)(k + u) * n + i, left, 0.f, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += v[u][e];
        }
        store_values<ACH_F32>(dw + i, left, s);
    }
}

bool fc_desc(const ach_fc_desc *d, ach_fc_desc *out)
{
    if (!d || d->rows < 0 || d->inputs < 1 || d->outputs < 1) return false;
    if (d->rows > KEPT_MOST || d->inputs > MOST_COLUMNS || d->outputs > MOST_COLUMNS) return false;
    if (!elem_type(d->type) || d->stride < 0) return false;
    *out = *d;
    if (out->stride == 0) out->stride = d->outputs;
    return out->stride >= d->outputs && out->stride <= MOST_COLUMNS;
}

struct Plan {
    int o, i;  // outputs and inputs of a tile: 128 x 128, 256 x 128 or 128 x 256
    int ti, to, span, slices;
    size_t bytes;
};

int tiles_of(int n, int tile) { return (n + tile - 1) / tile; }
int whole_turns(int stages) { return stages + stages % RING; }

Plan fc_plan(const ach_fc_desc &d)
{
    Plan p;
    const int stages = tiles_of(d.rows, DEPTH);
    // Small tiles, of which two workgroups run on a compute unit, one writing while the
    // other multiplies: on few rows (128 x 9216 -> 4096 fp32 45 us, 51 in large ones, bf16
    // 31 and 34; 256 rows fp32 69 and 73; 400 rows 105 and 107, bf16 54 and 52; 1000 x 4096
    // -> 4096 fp32 99 and 91), and on some more where they keep more of the compute units
    // busy without slices (600 x 2000 -> 1500 fp32 24 and 28, 1000 rows 34 and 32).
    const int64_t small = (int64_t)tiles_of(d.outputs, 128) * tiles_of(d.inputs, 128),
                  high = (int64_t)tiles_of(d.outputs, 256) * tiles_of(d.inputs, 128),
                  wide = (int64_t)tiles_of(d.outputs, 128) * tiles_of(d.inputs, 256);
    p.o = p.i = 128;
    if (stages > (small <= 256 ? 20 : 8)) {
        if (high < wide || (high == wide && d.type == ACH_BF16)) p.o = 256;
        else p.i = 256;
    }
    p.to = tiles_of(d.outputs, p.o);
    p.ti = tiles_of(d.inputs, p.i);
    const int64_t tiles = (int64_t)p.ti * p.to;
    // Up to 256 workgroups, each of four stages or more; as many as cost least, a stage
    // 0.85 us and the sums of the slices 3 us and their writing and reading: 300 x 2000 ->
    // 1500 fp32 19 us in one, 23 in two, 27 in three; 600 rows 28, 27, 32; 2000 x 4096 ->
    // 1000 bf16 42, 38 in two, 41 in three; 1531 x 1003 -> 777 fp16 49, 21 in six to nine.
    // Long bf16 deltas, from 256 stages of a slice on, two a compute unit: 512.  4096 ->
    // 1024 of 16384 rows 147 us, with up to 256 154; 12000 rows 114 and 117, 8192 86 and
    // 85, 6000 70 and 68 (2048 -> 2048 the same within a us).  Where 256 is not a multiple
    // of the tiles it gains more, and sooner: 9000 -> 500, 142 tiles, of 16384 rows 217 and
    // 373, 8192 118 and 190, 6000, which the rule leaves in 142 workgroups, 93 and 141.
    const size_t bytes = (size_t)d.outputs * d.inputs * sizeof(float);
    const int one_round = tiles < 256 ? (int)(256 / tiles) : 1;
    int each = whole_turns(stages), slices = one_round;
    if (d.type == ACH_BF16 && p.o == 256 && tiles < 512 && stages / one_round >= 256) {
        slices = min((int)(512 / tiles), MOST_SLICES);
        each = whole_turns(tiles_of(stages, slices));
    } else {
        slices = min(min(one_round, stages / 4), MOST_SLICES);
        size_t least = (size_t)each * 850;
        for (int n = 2; n <= slices; ++n) {
            const int e = whole_turns(tiles_of(stages, n));
            const size_t cost = (size_t)e * 850 + 3000 + n * (bytes / 4000);
            if (cost < least) least = cost, each = e;
        }
    }
    p.slices = each ? tiles_of(stages, each) : 1;
    p.span = each * DEPTH;
    p.bytes = p.slices > 1 ? p.slices * bytes : 0;
    return p;
}

template <int TYPE, int WO, int WI, int MO, int HOW>
int fc_launch(const Plan &p, const void *delta, const Fc &a, hipStream_t st)
{
    using S = Tile<TYPE, WO, WI, MO>;
    const auto kern = &k_fc_wgrad<TYPE, WO, WI, MO, HOW>;
    if (S::LDS > 64 * 1024) {
        const int rc = check(hipFuncSetAttribute(reinterpret_cast<const void *>(kern),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::LDS));
        if (rc) return rc;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.ti * p.to), (unsigned)p.slices), dim3(S::THREADS),
                       S::LDS, st, (const typename Elem<TYPE>::T *)delta, a);
    return check_launch();
}

template <int TYPE, int WO, int WI, int MO>
int fc_go(const Plan &p, const void *delta, const Fc &a, hipStream_t st)
{
    if constexpr (TYPE != ACH_F32) {
        if (a.outputs < 8) return fc_launch<TYPE, WO, WI, MO, SINGLE>(p, delta, a, st);
        if (a.outputs % 8) return fc_launch<TYPE, WO, WI, MO, EARLY>(p, delta, a, st);
    }
    return fc_launch<TYPE, WO, WI, MO, WHOLE>(p, delta, a, st);
}

// bf16 deltas, whose tiles cost the matrix units a third of the others' time, need
// fewer loads of operands from LDS: four waves of 128 x 64, two workgroups a
// compute unit.
template <int TYPE> int fc_tiles(const Plan &p, const void *delta, const Fc &a, hipStream_t st)
{
    if (p.i == 256) return fc_go<TYPE, 2, 4, 2>(p, delta, a, st);
    if (p.o == 128) return fc_go<TYPE, 2, 2, 2>(p, delta, a, st);
    if constexpr (TYPE == ACH_BF16) return fc_go<TYPE, 2, 2, 4>(p, delta, a, st);
    else return fc_go<TYPE, 4, 2, 2>(p, delta, a, st);
}

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_fc_bwd_filter_checkpoint_workspace(const ach_fc_desc *desc)
{
    ach_fc_desc d;
    return fc_desc(desc, &d) ? fc_plan(d).bytes : 0;
}

int ach_fc_bwd_filter_checkpoint(const ach_fc_desc *desc, const void *checkpoint, const void *delta,
                                 float *dw, int accumulate, void *ws, size_t ws_bytes,
                                 ach_stream_t s)
{
    ach_fc_desc d;
    if (!fc_desc(desc, &d) || !checkpoint || !delta || !dw) return ACH_EINVAL;
    if (accumulate != 0 && accumulate != 1) return ACH_EINVAL;
    if (!aligned(checkpoint, 16) || !aligned(delta, elem_size(d.type)) || !aligned(dw, 4))
        return ACH_EINVAL;
    const Plan p = fc_plan(d);
    if ((int64_t)p.ti * p.to >= 1 << 23) return ACH_EINVAL;  // more of dw than a card holds
    if (p.bytes && (!ws || ws_bytes < p.bytes || !aligned(ws, 16))) return ACH_EWORKSPACE;
    // dw of more than the L2 caches hold goes past them where its rows are whole lines
    // of 128 bytes (128 x 9216 -> 4096 fp32 51 us, 54 in them; 9000 inputs 60 and 59, bf16
    // 43 and 42, one row of it 43 and 34)
    const bool past = p.slices == 1 && d.inputs % 32 == 0 && aligned(dw, 128) &&
                      (size_t)d.outputs * d.inputs * sizeof(float) > (size_t)32 << 20;
    const Fc a = {d.rows, d.inputs, d.outputs, d.stride, kept(checkpoint, d.rows, d.inputs), dw,
                  p.slices > 1 ? (float *)ws : nullptr, accumulate, p.span, p.ti, past};
    hipStream_t st = as_stream(s);
    int rc;
#define CALL(TYPE) rc = fc_tiles<TYPE>(p, delta, a, st)
    FOR_TYPE(d.type, CALL);
#undef CALL
    if (rc || p.slices == 1) return rc;
    const size_t n = (size_t)d.outputs * d.inputs;
    hipLaunchKernelGGL(k_fc_wgrad_join, dim3(grid_for((n + 3) / 4, 256, 4096)), dim3(256), 0, st,
                       (const float *)ws, n, p.slices, dw, accumulate);
    return check_launch();
}

}  // extern "C"
