// Activation checkpoints in 8 bits (include/aetcnn_ops.h): pack and unpack.
//
// Bound by memory: a value is read and written once, a lane 16 bytes of it at a
// time, so that a block's 32 values lie in 4 (16-bit types) or 8 adjacent lanes,
// which find its largest magnitude by lane shifts.  All powers of two are put
// together from their exponents; products with them are exact.
#include "checkpoint.hpp"

namespace ach {
namespace {

constexpr int THREADS = 256;

// n chunks of `per` a row
template <int TYPE, bool PACK>
__global__ void __launch_bounds__(THREADS)
k_checkpoint(typename Elem<TYPE>::T *x, int64_t stride, int features, int n, FastDiv per, Kept k,
             bool past)
{
    constexpr int VEC = Row<TYPE>::VEC;
    // (a block's lanes stay together: n and the grid's step are multiples of their number)
    for (int64_t q = (int64_t)blockIdx.x * THREADS + threadIdx.x; q < n;
         q += (int64_t)gridDim.x * THREADS) {
        const int r = fdiv((int)q, per), col = ((int)q - r * (int)per.d) * VEC;
        typename Elem<TYPE>::T *p = x + r * stride + col;
        float v[VEC];
        if (PACK) {
            load_values<TYPE>(p, features - col, v);
            keep_values<VEC>(k, (size_t)q * VEC, v);
        } else {
            kept_values<VEC>(k, (size_t)q * VEC, v);
            if (TYPE == ACH_F16) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)  // 64 steps of 1024 are above the largest
                    v[i] = v[i] == v[i] ? __builtin_amdgcn_fmed3f(v[i], -65504.f, 65504.f) : v[i];
            }
            if (past) store_values<TYPE, true>(p, features - col, v);
            else store_values<TYPE>(p, features - col, v);
        }
    }
}

bool checkpoint_desc(const ach_checkpoint_desc *d, ach_checkpoint_desc *out)
{
    if (!d || d->rows < 0 || d->features < 1 || d->features > KEPT_MOST || d->stride < 0) return false;
    if (d->rows > KEPT_MOST || !elem_type(d->type)) return false;
    *out = *d;
    if (out->stride == 0) out->stride = d->features;
    return out->stride >= d->features;
}

template <int TYPE, bool PACK>
int go(const ach_checkpoint_desc &d, void *x, const void *checkpoint, hipStream_t st)
{
    constexpr int VEC = Row<TYPE>::VEC;
    using T = typename Elem<TYPE>::T;
    Kept k = kept(checkpoint, d.rows, d.features);
    const int per = k.width / VEC;
    const FastDiv div = make_fastdiv((unsigned)per);
    // values of more than the L2 caches hold go past them (128 x 290400 fp32, both
    // ways: 73 us, 64 past them)
    const bool past = (size_t)d.rows * d.features * sizeof(T) > (size_t)32 << 20;
    // launches of as many rows as have fewer than 2^31 chunks (a row: 2^28 at most)
    const int most = 0x7fffffff / per;
    for (int r = 0; r < d.rows; r += most) {
        const int rows = d.rows - r < most ? d.rows - r : most;
        const int n = rows * per;
        hipLaunchKernelGGL((k_checkpoint<TYPE, PACK>), dim3(grid_for((size_t)n, THREADS, 1u << 22)),
                           dim3(THREADS), 0, st, (T *)x + (size_t)r * d.stride, d.stride, d.features,
                           n, div, k, past);
        const int rc = check_launch();
        if (rc) return rc;
        k.codes += (size_t)rows * k.width;
        k.steps += (size_t)rows * (k.width / KEPT_BLOCK);
    }
    return ACH_OK;
}

template <bool PACK>
int checkpoint(const ach_checkpoint_desc *desc, const void *x, const void *checkpoint, ach_stream_t s)
{
    ach_checkpoint_desc d;
    if (!checkpoint_desc(desc, &d) || !x || !checkpoint) return ACH_EINVAL;
    if (!aligned(x, elem_size(d.type)) || !aligned(checkpoint, 16)) return ACH_EINVAL;
    if (d.rows == 0) return ACH_OK;
#define CALL(TYPE) return go<TYPE, PACK>(d, const_cast<void *>(x), checkpoint, as_stream(s))
    FOR_TYPE(d.type, CALL);
#undef CALL
}

}  // namespace
}  // namespace ach

using namespace ach;

extern "C" {

size_t ach_checkpoint_bytes(int rows, int features)
{
    if (rows < 0 || rows > KEPT_MOST || features < 1 || features > KEPT_MOST) return 0;
    const size_t blocks = ((size_t)features + KEPT_BLOCK - 1) / KEPT_BLOCK;
    return (size_t)rows * blocks * (KEPT_BLOCK + 1);
}

int ach_checkpoint_pack(const ach_checkpoint_desc *d, const void *x, void *checkpoint,
                        ach_stream_t stream)
{
    return ach::checkpoint<true>(d, x, checkpoint, stream);
}

int ach_checkpoint_unpack(const ach_checkpoint_desc *d, const void *checkpoint, void *x,
                          ach_stream_t stream)
{
    return ach::checkpoint<false>(d, x, checkpoint, stream);
}

}  // extern "C"
