// Reductions over a wave without LDS: rotations within rows of 16 lanes, then
// the rows and the halves by lane swaps.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

namespace vkv {

template <int BY> __device__ __forceinline__ float row_turn(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + BY, 0xf, 0xf, false));
}

// over the four 16-lane rows of a wave, lane by lane
template <typename F> __device__ __forceinline__ float rows_reduce(float x, F f) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <typename F> __device__ __forceinline__ float wave_reduce(float x, F f) {
    x = f(x, row_turn<8>(x));
    x = f(x, row_turn<4>(x));
    x = f(x, row_turn<2>(x));
    x = f(x, row_turn<1>(x));
    return rows_reduce(x, f);
}

struct Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
    __device__ float operator()(float a, float b) const { return a + b; }
};
__device__ __forceinline__ float wave_max(float x) { return wave_reduce(x, Max()); }
__device__ __forceinline__ float wave_sum(float x) { return wave_reduce(x, Sum()); }
__device__ __forceinline__ float rows_max(float x) { return rows_reduce(x, Max()); }
__device__ __forceinline__ float rows_sum(float x) { return rows_reduce(x, Sum()); }

}  // namespace vkv
