// Element access by run-time type (DDCN_F32 / DDCN_BF16 / DDCN_F16), values in fp32: shared by the optimizer and the 8-bit
// product.  gfx950 only.
#pragma once
#include "ddcn_16bit.h"

namespace ddcn {
namespace {

template <int DT> __device__ __forceinline__ float load_one(const void *p, long long i)
{
    if (DT == DDCN_F32) return ((const float *)p)[i];
    const bf16_t u = ((const bf16_t *)p)[i];
    return DT == DDCN_BF16 ? BF16::one(u) : F16::one(u);
}
template <int DT> __device__ __forceinline__ void load_four(const void *p, long long i, float (&x)[4])
{
    if (DT == DDCN_F32) {
        const f32x4 u = *(const f32x4 *)((const float *)p + i);
        for (int e = 0; e < 4; ++e) x[e] = u[e];
    } else {
        const uint2 u = *(const uint2 *)((const bf16_t *)p + i);
        x[0] = DT == DDCN_BF16 ? BF16::lo(u.x) : F16::lo(u.x);
        x[1] = DT == DDCN_BF16 ? BF16::hi(u.x) : F16::hi(u.x);
        x[2] = DT == DDCN_BF16 ? BF16::lo(u.y) : F16::lo(u.y);
        x[3] = DT == DDCN_BF16 ? BF16::hi(u.y) : F16::hi(u.y);
    }
}
template <int DT> __device__ __forceinline__ void store_one(void *p, long long i, float x)
{
    if (DT == DDCN_F32) ((float *)p)[i] = x;
    else ((bf16_t *)p)[i] = (bf16_t)(DT == DDCN_BF16 ? BF16::pack2(x, 0.f) : F16::pack2(x, 0.f));
}
template <int DT> __device__ __forceinline__ void store_four(void *p, long long i, const float (&x)[4])
{
    if (DT == DDCN_F32) {
        *(f32x4 *)((float *)p + i) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
        uint2 u;
        u.x = DT == DDCN_BF16 ? BF16::pack2(x[0], x[1]) : F16::pack2(x[0], x[1]);
        u.y = DT == DDCN_BF16 ? BF16::pack2(x[2], x[3]) : F16::pack2(x[2], x[3]);
        *(uint2 *)((bf16_t *)p + i) = u;
    }
}
// Four elements from i on, of which `live` exist (the others read 0); vec: the address allows one wide access
template <int DT> __device__ __forceinline__ void load_some(const void *p, long long i, int live, bool vec, float (&x)[4])
{
    if (vec && live >= 4) return load_four<DT>(p, i, x);
    for (int e = 0; e < 4; ++e) x[e] = e < live ? load_one<DT>(p, i + e) : 0.f;
}
template <int DT> __device__ __forceinline__ void store_some(void *p, long long i, int live, bool vec, const float (&x)[4])
{
    if (vec && live >= 4) return store_four<DT>(p, i, x);
    for (int e = 0; e < 4; ++e)
        if (e < live) store_one<DT>(p, i + e, x[e]);
}

}  // namespace
}  // namespace ddcn
