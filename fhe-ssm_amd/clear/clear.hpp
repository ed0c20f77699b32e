// clear.hpp -- what the kernels of libfhe_ssm_clear.so share: error reports, element types, wave sums.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "fhe_ssm_clear.h"

namespace clear {

// ---------------------------------------------------------------- host: status codes (nothing here throws)
char* error_text();  // this thread's message
constexpr size_t kErrorText = 512;

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(error_text(), kErrorText, fmt, ap);
    va_end(ap);
    return code;
}

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? CKKS_OK : fail(CKKS_EHIP, "%s: %s", what, hipGetErrorString(e));
}

inline size_t type_bytes(uint32_t type) { return type == FHE_SSM_F32 ? 4 : 2; }

inline bool aligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }

// ---------------------------------------------------------------- element types
typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <class T>
__device__ inline float to_f32(T x) {
    return (float)x;
}
template <>
__device__ inline float to_f32<bf16>(bf16 x) {
    return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, x) << 16);
}

// rounds to nearest even: the one rounding of an output
template <class T>
__device__ inline T from_f32(float x) {
    return (T)x;
}

// ---------------------------------------------------------------- sums over lanes, by row shifts and row broadcasts
template <int kControl, int kRows>
__device__ inline uint64_t moved(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, kControl, kRows, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), kControl, kRows, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
template <int kControl, int kRows, class T>
__device__ inline T plus_moved(T x) {
    return x + __builtin_bit_cast(T, moved<kControl, kRows>(__builtin_bit_cast(uint64_t, x)));
}
// lane l: the sum of lanes 0 .. l
template <class T>
__device__ inline T wave_scan(T x) {
    x = plus_moved<0x111, 0xf>(x);
    x = plus_moved<0x112, 0xf>(x);
    x = plus_moved<0x114, 0xf>(x);
    x = plus_moved<0x118, 0xf>(x);
    x = plus_moved<0x142, 0xa>(x);
    return plus_moved<0x143, 0xc>(x);
}
template <class T>
__device__ inline T from_lane(T x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}
template <class T>
__device__ inline T wave_sum(T x) {
    return from_lane(wave_scan(x), 63);
}
}  // namespace clear
