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
__device__ __forceinline__ void narrow(float v, Bf16 &out) { out.bits = __builtin_bit_cast(unsigned short, (__bf16)v); }

__device__ __forceinline__ float ninf(float) { return -__builtin_huge_valf(); }
__device__ __forceinline__ double ninf(double) { return -__builtin_huge_val(); }
__device__ __forceinline__ float nan_of(float) { return __builtin_nanf(""); }
__device__ __forceinline__ double nan_of(double) { return __builtin_nan(""); }

// op over all of a group of G lanes (a power of two, aligned), the same result in each.  Lanes meet their
// neighbours, quads, halves of a row of 16 and rows through the cross-lane paths of the vector unit; no LDS.
template <int CTRL>
__device__ __forceinline__ unsigned lane_move(unsigned v)
{
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int STEP, typename V>
__device__ __forceinline__ void lane_pair(V v, V &a, V &b)
{
    constexpr int N = sizeof(V) / 4;
    struct Words { unsigned w[N]; };
    const Words x = __builtin_bit_cast(Words, v);
    Words p, q;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (STEP == 32) {
            const auto r = __builtin_amdgcn_permlane32_swap(x.w[i], x.w[i], false, false);
            p.w[i] = r[0], q.w[i] = r[1];
        } else if constexpr (STEP == 16) {
            const auto r = __builtin_amdgcn_permlane16_swap(x.w[i], x.w[i], false, false);
            p.w[i] = r[0], q.w[i] = r[1];
        } else {
            p.w[i] = x.w[i];
            q.w[i] = lane_move<STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : STEP == 4 ? 0x141 : 0x140>(x.w[i]);
        }
    }
    a = __builtin_bit_cast(V, p);
    b = __builtin_bit_cast(V, q);
}
template <int G, typename V, typename Op>
__device__ __forceinline__ V over_lanes(V v, Op op)
{
    V a, b;
    if constexpr (G > 1) lane_pair<1>(v, a, b), v = op(a, b);
    if constexpr (G > 2) lane_pair<2>(v, a, b), v = op(a, b);
    if constexpr (G > 4) lane_pair<4>(v, a, b), v = op(a, b);
    if constexpr (G > 8) lane_pair<8>(v, a, b), v = op(a, b);
    if constexpr (G > 16) lane_pair<16>(v, a, b), v = op(a, b);
    if constexpr (G > 32) lane_pair<32>(v, a, b), v = op(a, b);
    return v;
}
template <int G, typename V>
__device__ __forceinline__ V lanes_max(V v)
{
    return over_lanes<G>(v, [](V a, V b) { return a > b ? a : b; });
}
template <int G, typename V>
__device__ __forceinline__ V lanes_sum(V v)
{
    return over_lanes<G>(v, [](V a, V b) { return a + b; });
}

// N consecutive elements in one access.  The type says only what a tensor guarantees (its element's
// alignment): a view into a flat buffer may start anywhere, and the hardware takes such addresses.
// What streams past once is read and written past the caches' order of use (nontemporal): of the loss over
// 4096 x 128000 bf16 logits both together took 606 us to 501, the step with 8-bit moments 593 to 462.
template <typename T, int N>
struct Pack {
    T v[N];
};
template <int BYTES> struct Words;
template <> struct Words<4> { typedef unsigned type __attribute__((aligned(2))); };
template <> struct Words<8> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Words<16> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Words<32> { typedef unsigned type __attribute__((ext_vector_type(8), aligned(2))); };

template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p)
{
    typedef typename Words<sizeof(Pack<T, N>)>::type V;
    const V w = __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
    Pack<T, N> r;
    __builtin_memcpy(&r, &w, sizeof(r));
    return r;
}
template <int N, typename T>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r)
{
    typedef typename Words<sizeof(Pack<T, N>)>::type V;
    V w;
    __builtin_memcpy(&w, &r, sizeof(r));
    __builtin_nontemporal_store(w, reinterpret_cast<V *>(p));
}
// N elements at p + k of a tensor of n, zeros behind its end.
template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load_some(const T *p, long k, long n)
{
    if (k + N <= n) return load_pack<N>(p + k);
    Pack<T, N> r = {};
#pragma unroll
    for (int e = 0; e < N; e++)
        if (k + e < n) r.v[e] = p[k + e];
    return r;
}
template <int N, typename T>
__device__ __forceinline__ void store_some(T *p, long k, long n, const Pack<T, N> &r)
{
    if (k + N <= n) {
        store_pack<N>(p + k, r);
        return;
    }
#pragma unroll
    for (int e = 0; e < N; e++)
        if (k + e < n) p[k + e] = r.v[e];
}
#endif

}  // namespace ccnn
