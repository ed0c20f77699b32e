// rows.hpp -- rows of 32- or 16-bit elements taken as float32 by a few lanes, a wave or a workgroup, and sums over them.
#pragma once
#include "clear.hpp"

namespace clear {

// f(an element of the type), whose value says nothing
template <class F>
auto by_type(uint32_t type, F&& f) {
    return type == FHE_SSM_F32 ? f(0.f) : type == FHE_SSM_BF16 ? f(bf16{}) : f(f16{});
}

// V elements at p, which lies on their size
template <int V, class T>
__device__ inline void load(const T* p, float* f) {
    if constexpr (V == 1) {
        f[0] = to_f32(*p);
    } else {
        typedef T vec __attribute__((ext_vector_type(V)));
        const vec v = *(const vec*)p;
#pragma unroll
        for (int c = 0; c < V; c++) f[c] = to_f32((T)v[c]);
    }
}
template <int V, class T>
__device__ inline void store(T* p, const float* f) {
    if constexpr (V == 1) {
        *p = from_f32<T>(f[0]);
    } else {
        typedef T vec __attribute__((ext_vector_type(V)));
        vec v;
#pragma unroll
        for (int c = 0; c < V; c++) v[c] = from_f32<T>(f[c]);
        *(vec*)p = v;
    }
}

template <int kControl>
__device__ inline float swapped(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kControl, 0xf, 0xf, false));
}
// the sum over each 16 lanes, the same in all of them: neighbours, pairs, fours, eights.  (A product summed would be rounded
// for the other lanes and not for its own, if the addition took it in.)
__device__ inline float sum16(float x) {
#pragma clang fp contract(off)
    x += swapped<0xb1>(x);
    x += swapped<0x4e>(x);
    x += swapped<0x141>(x);
    return x + swapped<0x140>(x);
}
__device__ inline float of_lane(float x, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(x), lane));
}
__device__ inline float sum64(float x) {
    x = sum16(x);
    return (of_lane(x, 0) + of_lane(x, 16)) + (of_lane(x, 32) + of_lane(x, 48));
}

// the largest of each 16 lanes, of the wave, in all of them; a NaN is none
__device__ inline float max16(float x) {
    x = __builtin_fmaxf(x, swapped<0xb1>(x));
    x = __builtin_fmaxf(x, swapped<0x4e>(x));
    x = __builtin_fmaxf(x, swapped<0x141>(x));
    return __builtin_fmaxf(x, swapped<0x140>(x));
}
__device__ inline float max64(float x) {
    x = max16(x);
    return __builtin_fmaxf(__builtin_fmaxf(of_lane(x, 0), of_lane(x, 16)), __builtin_fmaxf(of_lane(x, 32), of_lane(x, 48)));
}

// N sums over the L lanes that share a row, in all of them and always in the same order.  L of 256 or 1,024 is the workgroup:
// the waves' sums go through LDS, two blocks of them in turn, so that one barrier is enough.
template <int L, int N>
struct Sums {
    static constexpr int kWaves = L < 64 ? 1 : L / 64;
    float part[2][N][kWaves];
};
template <int L, int N>
__device__ inline void sum_over(float (&x)[N], Sums<L, N>& s, int turn) {
    if constexpr (L == 16) {
#pragma unroll
        for (int n = 0; n < N; n++) x[n] = sum16(x[n]);
    } else {
#pragma unroll
        for (int n = 0; n < N; n++) x[n] = sum64(x[n]);
    }
    if constexpr (L > 64) {
        constexpr int kWaves = L / 64;
        static_assert(kWaves <= 16);
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int n = 0; n < N; n++) s.part[turn][n][threadIdx.x / 64] = x[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; n++)
            x[n] = of_lane(sum16(threadIdx.x % 16 < kWaves ? s.part[turn][n][threadIdx.x % 16] : 0.f), 0);
    }
}

}  // namespace clear
