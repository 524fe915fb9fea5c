// A fully connected layer's weight gradient from its input's 8-bit checkpoint
// (include/aetcnn_ops.h).
#include "checkpoint.hpp"

namespace ach {
namespace {

constexpr int TILE = 64, DEPTH = 16;

struct Fc {
    int rows, inputs, outputs;
    int64_t stride;
    Kept k;
    float *dw;
    int accumulate;
};

// 64 x 64 of dw a workgroup, 4 x 4 a thread, 16 rows at a time through LDS
template <int TYPE>
__global__ void __launch_bounds__(256) k_fc_wgrad(const typename Elem<TYPE>::T *delta, Fc a)
{
    __shared__ float sd[DEPTH][TILE], sx[DEPTH][TILE];
    const int tiles = (a.inputs + TILE - 1) / TILE;
    const int o0 = (int)(blockIdx.x / tiles) * TILE, i0 = (int)(blockIdx.x % tiles) * TILE;
    const int to = threadIdx.x / 16 * 4, ti = threadIdx.x % 16 * 4;
    float acc[4][4] = {};
    for (int r0 = 0; r0 < a.rows; r0 += DEPTH) {
        for (int e = threadIdx.x; e < DEPTH * TILE; e += 256) {
            const int r = r0 + e / TILE, c = e % TILE;
            const bool there = r < a.rows;
            sd[e / TILE][c] = there && o0 + c < a.outputs ? (float)delta[r * a.stride + o0 + c] : 0.f;
            float v = 0.f;
            if (there && i0 + c < a.inputs) {
                const size_t at = (size_t)r * a.k.width + i0 + c;
                v = (float)a.k.codes[at] * kept_scale(a.k.steps[at / KEPT_BLOCK]);
            }
            sx[e / TILE][c] = v;
        }
        __syncthreads();
        for (int q = 0; q < DEPTH; ++q)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[u][v] += sd[q][to + u] * sx[q][ti + v];
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (o0 + to + u < a.outputs && i0 + ti + v < a.inputs) {
                float *p = a.dw + (size_t)(o0 + to + u) * a.inputs + i0 + ti + v;
                *p = a.accumulate ? *p + acc[u][v] : acc[u][v];
            }
}

bool fc_desc(const ach_fc_desc *d, ach_fc_desc *out)
{
    if (!d || d->rows < 0 || d->inputs < 1 || d->inputs > KEPT_MOST || d->outputs < 1) return false;
    if (!elem_type(d->type) || d->stride < 0) return false;
    *out = *d;
    if (out->stride == 0) out->stride = d->outputs;
    return out->stride >= d->outputs;
}

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_fc_bwd_filter_checkpoint_workspace(const ach_fc_desc *)
{
    return 0;
}

int ach_fc_bwd_filter_checkpoint(const ach_fc_desc *desc, const void *checkpoint, const void *delta,
                                 float *dw, int accumulate, void *, size_t, ach_stream_t s)
{
    ach_fc_desc d;
    if (!fc_desc(desc, &d) || !checkpoint || !delta || !dw) return ACH_EINVAL;
    if (accumulate != 0 && accumulate != 1) return ACH_EINVAL;
    if (!aligned(checkpoint, 16) || !aligned(delta, elem_size(d.type)) || !aligned(dw, 4))
        return ACH_EINVAL;
    const Fc a = {d.rows, d.inputs, d.outputs, d.stride, kept(checkpoint, d.rows, d.inputs), dw,
                  accumulate};
    const int64_t tiles = (int64_t)((d.inputs + TILE - 1) / TILE) * ((d.outputs + TILE - 1) / TILE);
    if (tiles > 0x7fffffff) return ACH_EUNSUPPORTED;
#define CALL(TYPE)                                                                                 \
    hipLaunchKernelGGL((k_fc_wgrad<TYPE>), dim3((unsigned)tiles), dim3(256), 0, as_stream(s),      \
                       (const Elem<TYPE>::T *)delta, a)
    FOR_TYPE(d.type, CALL);
#undef CALL
    return check_launch();
}

}  // extern "C"
