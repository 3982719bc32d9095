// nnsp_seq_dev.h -- device helpers of the sequence operators: loads and stores
// of the three element types at their natural alignment, cross-lane sums.
#ifndef NNSP_SEQ_DEV_H
#define NNSP_SEQ_DEV_H
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef float f32x4 __attribute__((ext_vector_type(4)));

// N elements at T's own alignment: global memory takes dword accesses at any
// byte address here, so a row that starts anywhere is still read 16 bytes a lane.
template <class T, int N>
struct Vec {
    typedef T raw __attribute__((ext_vector_type(N)));
    typedef raw type __attribute__((aligned(sizeof(T))));
};

template <class T, int N>
__device__ __forceinline__ void load_raw(T (&d)[N], const T* p) {
    const typename Vec<T, N>::type v = *reinterpret_cast<const typename Vec<T, N>::type*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = v[i];
}

template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&s)[N]) {
    typename Vec<T, N>::raw v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)s[i];
    *reinterpret_cast<typename Vec<T, N>::type*>(p) = v;
}

// lanes l and l ^ 8, l ^ 16, l ^ 32: rotation by half a row, then the two swaps
__device__ __forceinline__ float add_xor8(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_xor16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_xor32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// lanes l ^ 1, l ^ 2 (quad permutations), l ^ 4 (half-row mirror after the quads are equal)
__device__ __forceinline__ float add_xor1(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xb1, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_xor2(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4e, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_mirror4(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, true));
}
// sum over groups of W consecutive lanes (8, 16, 32, 64), in every lane
template <int W>
__device__ __forceinline__ float lane_sum(float x) {
    x = add_mirror4(add_xor2(add_xor1(x)));
    if (W >= 16) x = add_xor8(x);
    if (W >= 32) x = add_xor16(x);
    if (W >= 64) x = add_xor32(x);
    return x;
}

// exp(g) of a decay's logarithm.  Everything at or below -128 is 0 in 32 bits
// either way (exp(-104) is), and -infinity stays out of later differences.
__device__ __forceinline__ float decay_log(float g) { return g < -128.0f ? -128.0f : g; }

#endif
