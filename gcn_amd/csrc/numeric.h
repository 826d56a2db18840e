// Element types of the scoring and optimiser kernels (score.hip, adamw.hip): how each is read, written
// and widened.  Arithmetic is done in Wide<T>: fp32 for the 32- and 16-bit types, fp64 for doubles.
#pragma once
#include "ccnn_common.h"

namespace ccnn {

inline int type_bytes(int type)
{
    return type == CCNN_TYPE_F64 ? 8 : type == CCNN_TYPE_F32 ? 4 : type == CCNN_TYPE_BF16 || type == CCNN_TYPE_F16 ? 2 : 0;
}

#ifdef __HIPCC__
struct Bf16 { unsigned short bits; };
typedef _Float16 F16;

template <typename T> struct WideOf { typedef float type; };
template <> struct WideOf<double> { typedef double type; };
template <typename T> using Wide = typename WideOf<T>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(F16 v) { return (float)v; }
__device__ __forceinline__ float widen(Bf16 v) { return __uint_as_float((unsigned)v.bits << 16); }

// Rounded to nearest, ties to even: the one rounding of a 16-bit result.
__device__ __forceinline__ void narrow(float v, float &out) { out = v; }
__device__ __forceinline__ void narrow(double v, double &out) { out = v; }
__device__ __forceinline__ void narrow(float v, F16 &out) { out = (F16)v; }
__device__ __forceinline__ void narrow(float v, Bf16 &out)
{
    const unsigned u = __float_as_uint(v);
    out.bits = v != v ? 0x7fc0 : (unsigned short)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
}

__device__ __forceinline__ float ninf(float) { return -__builtin_huge_valf(); }
__device__ __forceinline__ double ninf(double) { return -__builtin_huge_val(); }
__device__ __forceinline__ float nan_of(float) { return __builtin_nanf(""); }
__device__ __forceinline__ double nan_of(double) { return __builtin_nan(""); }

// N consecutive elements in one access.  The type says only what a tensor guarantees (its element's
// alignment): a view into a flat buffer may start anywhere, and the hardware takes such addresses.
template <typename T, int N>
struct Pack {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p)
{
    Pack<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r)
{
    __builtin_memcpy(p, &r, sizeof(r));
}
#endif

}  // namespace ccnn
