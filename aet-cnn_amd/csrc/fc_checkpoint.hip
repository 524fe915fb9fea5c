// A fully connected layer's weight gradient from its input's 8-bit checkpoint
// (include/aetcnn_ops.h): dw = delta^T x on the bf16 matrix instructions.
//
// A code times its power of two is a bf16 number, and so is each piece of a
// delta (its first 8 bits, the next 8, the last 8; one piece for bf16, two for
// fp16, three for fp32): every product is exact and is summed in fp32.
//
// Tiles of 128 outputs x 128 inputs, a wave 64 x 64 of it.  A stage of 32 rows
// of both operands is loaded two stages ahead, turned into bf16 and stored as it
// lies in memory, [row][128]; the matrix instructions want 8 rows of a column in
// a lane, which the transposing LDS loads give: 16 lanes read 4 rows x 16
// columns, and each gets a column of it.
#include "checkpoint.hpp"
#include "pieces.hpp"

namespace ach {
namespace {

constexpr int TILE = 128, DEPTH = 32;
constexpr int PITCH = TILE + 32;  // 16-bit values of an LDS row
constexpr int MOST_SLICES = 64;

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
    int ti, to;        // tiles along the inputs and the outputs
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

// Eight values of a delta as pieces whose sum they are.
template <int TYPE> struct Eight {
    using T = typename Elem<TYPE>::T;
    float f[8];
    __device__ __forceinline__ void load(const T *p, int left)
    {
        if (left >= 8) {
            const typename Row<TYPE>::Chunk a = Row<TYPE>::load(p);
#pragma unroll
            for (int i = 0; i < Row<TYPE>::VEC; ++i) f[i] = (float)a[i];
            if constexpr (TYPE == ACH_F32) {
                const typename Row<TYPE>::Chunk b = Row<TYPE>::load(p + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[4 + i] = b[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = i < left ? (float)p[i] : 0.f;
        }
    }
    __device__ __forceinline__ void split(v4u *p)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = f[2 * i], b = f[2 * i + 1];
#pragma unroll
            for (int q = 0; q < Pieces<TYPE>::N; ++q) {
                p[q][i] = upper_halves(a, b);
                a = below(a), b = below(b);
            }
        }
    }
};

// Eight columns of a tile in LDS as a lane's operand of a 16-row step: `p` is
// the lane's own place in the first four rows.
__device__ __forceinline__ v8bf fragment(const short *p)
{
    typedef __attribute__((address_space(3))) v4s *Lds;
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p),
              b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * PITCH));
    const v8s v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(v8bf, v);
}

template <int TYPE>
__global__ void __launch_bounds__(256, 2) k_fc_wgrad(const typename Elem<TYPE>::T *delta, Fc a)
{
    constexpr int P = Pieces<TYPE>::N;
    __shared__ __align__(16) short sm[2][P + 1][DEPTH * PITCH];  // pieces of delta, then x
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wo = wave & 1, wi = wave >> 1;
    // each XCD, which takes every eighth workgroup, gets a contiguous range of
    // tiles, in groups of 8 outputs' tiles: they share the operands in its L2
    int id = blockIdx.x;
    {
        const int G = gridDim.x, g8 = G >> 3, r8 = G & 7, xcd = id & 7;
        id = xcd * g8 + min(xcd, r8) + (id >> 3);
    }
    const int group = id / (8 * a.ti), in = id - group * 8 * a.ti;
    const int high = min(8, a.to - group * 8);
    const int o0 = (group * 8 + in % high) * TILE, i0 = in / high * TILE;
    const int r0 = (int)blockIdx.y * a.span, r1 = min((int64_t)a.rows, (int64_t)r0 + a.span);

    // a thread's share of a stage: 16 codes of one row; 8 values of two rows
    const int xr = tid >> 3, xc = (tid & 7) * 16, dr = tid >> 4, dc = (tid & 15) * 8;
    const bool x_in = i0 + xc < a.k.width;
    const int d_left = a.outputs - (o0 + dc);
    v4u codes;
    uint32_t step;
    Eight<TYPE> d[2];
    auto load = [&](int r) {
        codes = 0;
        step = 7;
        if (r + xr < r1 && x_in) {
            const size_t at = (size_t)(r + xr) * a.k.width + i0 + xc;
            codes = *(const v4u *)(a.k.codes + at);
            step = a.k.steps[at / KEPT_BLOCK];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            d[h].load(delta + (r + dr + 16 * h) * a.stride + o0 + dc, r + dr + 16 * h < r1 ? d_left : 0);
    };
    auto store = [&](int s) {
        const float scale = kept_scale(step);
        v4u w[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float f[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) f[b] = (float)(int8_t)(codes[i] >> (8 * b)) * scale;
            w[i / 2][i % 2 * 2] = upper_halves(f[0], f[1]);
            w[i / 2][i % 2 * 2 + 1] = upper_halves(f[2], f[3]);
        }
        short *const to = &sm[s][P][xr * PITCH + xc];
        *(v4u *)to = w[0];
        *(v4u *)(to + 8) = w[1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4u p[P];
            d[h].split(p);
#pragma unroll
            for (int q = 0; q < P; ++q) *(v4u *)&sm[s][q][(dr + 16 * h) * PITCH + dc] = p[q];
        }
    };

    v16f hi[2][2], lo[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) hi[i][j][e] = lo[i][j][e] = 0.f;

    // a lane's place: rows 8 * (lane / 32) + lane % 16 / 4, columns 16 * (lane / 16 % 2) + 4 * (lane % 4)
    const int place = (8 * (lane >> 5) + ((lane & 15) >> 2)) * PITCH + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    load(r0);
    store(0);
    load(r0 + DEPTH);
    __syncthreads();
    int s = 0;
    for (int r = r0; r < r1; r += DEPTH, s ^= 1) {
#pragma unroll
        for (int step16 = 0; step16 < DEPTH / 16; ++step16) {
            v8bf x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                x[j] = fragment(&sm[s][P][place + step16 * 16 * PITCH + wi * 64 + j * 32]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v8bf p[P];
#pragma unroll
                for (int q = 0; q < P; ++q)
                    p[q] = fragment(&sm[s][q][place + step16 * 16 * PITCH + wo * 64 + i * 32]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    hi[i][j] = MFMA_BF(p[0], x[j], hi[i][j]);
#pragma unroll
                    for (int q = 1; q < P; ++q) lo[i][j] = MFMA_BF(p[q], x[j], lo[i][j]);
                }
            }
        }
        store(s ^ 1);  // (past the last stage: zeros, which nothing reads)
        load(r + 2 * DEPTH);
        __syncthreads();
    }
    float *const out = a.part ? a.part + (size_t)blockIdx.y * a.outputs * a.inputs : a.dw;
    const bool add = a.accumulate && !a.part;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int o = o0 + wo * 64 + i * 32 + 4 * (lane >> 5), c = i0 + wi * 64 + j * 32 + (lane & 31);
            if (c >= a.inputs) continue;
            float *const p = out + (size_t)o * a.inputs + c;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = 8 * (e >> 2) + (e & 3);
                if (o + r >= a.outputs) continue;
                float v = hi[i][j][e] + lo[i][j][e];
                if (add) v += p[(size_t)r * a.inputs];
                p[(size_t)r * a.inputs] = v;
            }
        }
}

__global__ void __launch_bounds__(256)
k_fc_wgrad_join(const float *part, size_t n, int slices, float *dw, int accumulate)
{
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float s = accumulate ? dw[i] : 0.f;
        for (int k = 0; k < slices; ++k) s += part[k * n + i];
        dw[i] = s;
    }
}

bool fc_desc(const ach_fc_desc *d, ach_fc_desc *out)
{
    if (!d || d->rows < 0 || d->inputs < 1 || d->inputs > KEPT_MOST || d->outputs < 1) return false;
    if (d->rows > KEPT_MOST) return false;
    if (!elem_type(d->type) || d->stride < 0) return false;
    *out = *d;
    if (out->stride == 0) out->stride = d->outputs;
    return out->stride >= d->outputs;
}

// Slices of the rows, so that two workgroups a compute unit run, of at least
// four stages each.
struct Plan {
    int ti, to, span, slices;
    size_t bytes;
};

Plan fc_plan(const ach_fc_desc &d)
{
    Plan p;
    p.ti = (int)(((int64_t)d.inputs + TILE - 1) / TILE);
    p.to = (int)(((int64_t)d.outputs + TILE - 1) / TILE);
    const int64_t tiles = (int64_t)p.ti * p.to;
    int slices = tiles < 512 ? (int)((511 + tiles) / tiles) : 1;
    const int stages = d.rows / DEPTH + (d.rows % DEPTH != 0);
    if (slices > stages / 4) slices = stages / 4;
    if (slices > MOST_SLICES) slices = MOST_SLICES;
    if (slices < 1) slices = 1;
    const int each = (stages + slices - 1) / slices;
    p.slices = each ? (stages + each - 1) / each : 1;
    p.span = each < 0x7fffffff / DEPTH ? each * DEPTH : 0x7fffffff;
    p.bytes = p.slices > 1 ? (size_t)p.slices * d.outputs * d.inputs * sizeof(float) : 0;
    return p;
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
    if ((int64_t)p.ti * p.to > 0x7fffffff) return ACH_EUNSUPPORTED;
    if (p.bytes && (!ws || ws_bytes < p.bytes || !aligned(ws, 16))) return ACH_EWORKSPACE;
    const Fc a = {d.rows, d.inputs, d.outputs, d.stride, kept(checkpoint, d.rows, d.inputs), dw,
                  p.slices > 1 ? (float *)ws : nullptr, accumulate, p.span, p.ti, p.to};
    hipStream_t st = as_stream(s);
#define CALL(TYPE)                                                                                 \
    hipLaunchKernelGGL((k_fc_wgrad<TYPE>), dim3((unsigned)(p.ti * p.to), (unsigned)p.slices),      \
                       dim3(256), 0, st, (const Elem<TYPE>::T *)delta, a)
    FOR_TYPE(d.type, CALL);
#undef CALL
    const int rc = check_launch();
    if (rc || p.slices == 1) return rc;
    const size_t n = (size_t)d.outputs * d.inputs;
    hipLaunchKernelGGL(k_fc_wgrad_join, dim3(grid_for(n, 256, 4096)), dim3(256), 0, st,
                       (const float *)ws, n, p.slices, dw, accumulate);
    return check_launch();
}

}  // extern "C"
