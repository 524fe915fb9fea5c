// Activations kept in 8 bits: the layout of a checkpoint and the arithmetic of
// its blocks (include/aetcnn_ops.h).
#pragma once

#include "rows.hpp"

namespace ach {

constexpr int KEPT_BLOCK = 32;

struct Kept {
    int8_t *codes;   // [rows][width]
    uint8_t *steps;  // [rows][width / KEPT_BLOCK]
    int width;       // features rounded up to whole blocks
};

inline Kept kept(const void *checkpoint, int rows, int features)
{
    Kept k;
    k.width = (features + KEPT_BLOCK - 1) / KEPT_BLOCK * KEPT_BLOCK;
    k.codes = (int8_t *)const_cast<void *>(checkpoint);
    k.steps = (uint8_t *)(k.codes + (size_t)rows * k.width);
    return k;
}
constexpr int KEPT_MOST = 1 << 30;  // rows and features

// The step of a block from the bits of its largest magnitude a: the biased
// exponent of a, whose power of two is 64 steps, or one more where a is 127.5
// steps or above (its mantissa is then 127/128 or above); 255 for a NaN or an
// infinity.
__device__ __forceinline__ uint32_t kept_step(uint32_t top)
{
    const uint32_t s = min(max((top + 0x10000u) >> 23, 7u), 254u);
    return top >= 0x7f800000u ? 255u : s;
}
// 2^(133 - step); 0 for step 255
__device__ __forceinline__ float kept_inverse(uint32_t step)
{
    return __uint_as_float(step == 255u ? 0u : (260u - step) << 23);
}
// 2^(step - 133); NaN for step 255
__device__ __forceinline__ float kept_scale(uint32_t step)
{
    return __uint_as_float(step == 255u ? 0x7fc00000u : (step - 6u) << 23);
}
// The code of x as the low byte of a float: the sum with 1.5 * 2^23 rounds to
// whole numbers, to nearest even.
__device__ __forceinline__ uint32_t kept_code(float x, float inverse)
{
    const float c = __builtin_amdgcn_fmed3f(x * inverse, -127.f, 127.f);
    return __float_as_uint(c + 0x1.8p23f);
}
__device__ __forceinline__ uint32_t kept_codes(const float *x, float inverse)
{
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (kept_code(x[i], inverse) & 0xffu) << (8 * i);
    return r;
}
// The largest magnitude among VEC values of each of 32 / VEC adjacent lanes.
template <int VEC> __device__ __forceinline__ uint32_t kept_top(const float *v)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    // lanes 1 and 2 apart, then the mirror image within eight lanes
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));
    if (VEC == 4) m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));
    return m;
}
// VEC values at `at` (a multiple of VEC) of the checkpoint's codes, by the 32 / VEC
// lanes of a block together.
template <int VEC>
__device__ __forceinline__ void keep_values(const Kept &k, size_t at, const float *v)
{
    const uint32_t step = kept_step(kept_top<VEC>(v));
    const float inverse = kept_inverse(step);
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) w[i] = kept_codes(v + 4 * i, inverse);
    __builtin_memcpy(__builtin_assume_aligned(k.codes + at, VEC), w, VEC);
    if (at % KEPT_BLOCK == 0) k.steps[at / KEPT_BLOCK] = (uint8_t)step;
}
// ... and back
template <int VEC>
__device__ __forceinline__ void kept_values(const Kept &k, size_t at, float *v)
{
    uint32_t w[VEC / 4];
    __builtin_memcpy(w, __builtin_assume_aligned(k.codes + at, VEC), VEC);
    const float scale = kept_scale(k.steps[at / KEPT_BLOCK]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
}

}  // namespace ach
