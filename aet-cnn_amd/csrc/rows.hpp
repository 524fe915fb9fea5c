// What the operators on rows of values of several types share (logits,
// layer norm, checkpoints): element types, loads, reductions over a wave.
#pragma once

#include "common.hpp"

namespace ach {

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
    // PAST the caches: for gradients that these would not hold until they are read
    template <bool PAST> static __device__ __forceinline__ void store(T *p, Chunk v)
    {
        if (PAST) __builtin_nontemporal_store(v, (Chunk *)p);
        else *(Chunk *)p = v;
    }
};

// A chunk's values as floats, of which `left` are there (the others: 0).
template <int TYPE>
__device__ __forceinline__ void load_values(const typename Elem<TYPE>::T *p, int left, float *v)
{
    constexpr int VEC = Row<TYPE>::VEC;
    if (left >= VEC) {
        const typename Row<TYPE>::Chunk c = Row<TYPE>::load(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = (float)c[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = i < left ? (float)p[i] : 0.f;
    }
}
template <int TYPE, bool PAST = false>
__device__ __forceinline__ void store_values(typename Elem<TYPE>::T *p, int left, const float *v)
{
    using T = typename Elem<TYPE>::T;
    constexpr int VEC = Row<TYPE>::VEC;
    if (left >= VEC) {
        typename Row<TYPE>::Chunk c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) c[i] = (T)v[i];
        Row<TYPE>::template store<PAST>(p, c);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}
// N floats of a row of parameters, of which `left` are there (the others: 0);
// `none` where there is no row.
template <int N>
__device__ __forceinline__ void load_floats(const float *p, size_t at, int left, float none, float *v)
{
    if (!p) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = none;
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i += 4) load_values<ACH_F32>(p + at + i, left - i, v + i);
}

// Sums over a wave without the LDS crossbar: within rows of 16 lanes by
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
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp(double v)
{
    const uint64_t u = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false),
              hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}
__device__ __forceinline__ double wave_total(double v)  // in lane 63 alone
{
    v += dpp<0x111, 0xf>(v);
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xa>(v);
    v += dpp<0x143, 0xc>(v);
    return v;
}
inline size_t elem_size(int type) { return type == ACH_F32 ? 4 : 2; }
inline bool elem_type(int type) { return type == ACH_F32 || type == ACH_BF16 || type == ACH_F16; }
inline bool aligned(const void *p, size_t size) { return ((uintptr_t)p & (size - 1)) == 0; }

}  // namespace ach

// CALL(TYPE) for the element type of a descriptor
#define FOR_TYPE(type, CALL)                                                                      \
    do {                                                                                          \
        if ((type) == ACH_F32) CALL(ACH_F32);                                                     \
        else if ((type) == ACH_BF16) CALL(ACH_BF16);                                              \
        else CALL(ACH_F16);                                                                       \
    } while (0)
