// Shared by the kernels of block-sparse attention: 16- and 8-bit element types, and how operands are described.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace lapis {

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// bf16 <-> f32: widening is exact, narrowing rounds to nearest even (one instruction on gfx950).
struct Bf16 {
  typedef __bf16 elem;
};
struct F16 {
  typedef _Float16 elem;
};

template <typename T>
using vec8 = typename T::elem __attribute__((ext_vector_type(8)));
template <typename T>
using vec4 = typename T::elem __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ void widen(vec8<T> x, float *f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)x[i];
}
template <typename T>
__device__ __forceinline__ vec8<T> narrow(const float *f) {
  vec8<T> x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (typename T::elem)f[i];
  return x;
}

// e4m3 codes (no infinities, largest 448, NaN 0x7f): eight to and from eight floats, rounding to nearest even
__device__ __forceinline__ void widen_f8(v2i x, float *f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(x[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x[i], true);
    f[4 * i] = lo[0], f[4 * i + 1] = lo[1], f[4 * i + 2] = hi[0], f[4 * i + 3] = hi[1];
  }
}
__device__ __forceinline__ v2i narrow_f8(const float *f) {
  v2i x = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], x[i], false);
    x[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], x[i], true);
  }
  return x;
}

// Maximum over aligned groups of W lanes, unsigned: of the bits of absolute values NaN is the largest.
template <int W>
__device__ __forceinline__ unsigned group_max(unsigned v) {
  if (W >= 2) v = max(v, (unsigned)dpp_mov<0xB1>((int)v));
  if (W >= 4) v = max(v, (unsigned)dpp_mov<0x4E>((int)v));
  if (W >= 8) v = max(v, (unsigned)dpp_mov<0x141>((int)v));
  if (W >= 16) v = max(v, (unsigned)dpp_mov<0x140>((int)v));
  if (W >= 32) v = max(v, (unsigned)__shfl_xor((int)v, 16, 64));
  if (W >= 64) v = max(v, (unsigned)__shfl_xor((int)v, 32, 64));
  return v;
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }
constexpr unsigned kInfBits = 0x7f800000u;

// ---- host: what every entry point asks of its operands --------------------------------------------------------

constexpr int kMaxDim = 256;       // of the cache and its attention
constexpr int kMaxBlockDim = 128;  // of block attention

int check_cache(const char *what, const lapis_hip_kv_cache *cache);

inline bool is_16bit(int dtype) { return dtype == LAPIS_HIP_BF16 || dtype == LAPIS_HIP_F16; }
inline bool strides_of_8(const int64_t *s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 8 != 0) return false;
  return true;
}

}  // namespace lapis
