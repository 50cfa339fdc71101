// A paged cache as kernels see it, and how eight elements of a row go into it and come out: 16 bits, 8-bit or 4-bit codes.
#pragma once
#include "attn.hpp"

namespace lapis {

enum Codes { kNoCodes = 0, kF8 = 1, kF4 = 2 };  // what a cache holds
inline Codes codes_of(int dtype) { return dtype == LAPIS_HIP_F8E4M3 ? kF8 : dtype == LAPIS_HIP_F4E2M1 ? kF4 : kNoCodes; }

struct CacheView {
  char *data[2];
  void *scale[2];
  long long stride[3], scale_stride[3];
  long long slots;  // pages * page
  int heads, page_log2, dim;
};
struct RowsView {
  char *data[2];
  long long stride[2][2];  // token, head
};

inline CacheView view_of(const lapis_hip_kv_cache *c) {
  CacheView v = {};
  v.data[0] = static_cast<char *>(c->k);
  v.data[1] = static_cast<char *>(c->v);
  v.scale[0] = c->k_scale;
  v.scale[1] = c->v_scale;
  for (int i = 0; i < 3; ++i) {
    v.stride[i] = c->stride[i];
    v.scale_stride[i] = c->scale_stride[i];
  }
  v.slots = c->pages * c->page;
  v.heads = c->heads;
  v.page_log2 = __builtin_ctz((unsigned)c->page);
  v.dim = c->dim;
  return v;
}

// Division of numbers below 2^31 by one that the host knows: q = r * m / 2^p, where p = 31 + ceil(log2 d) and m = ceil(2^p / d).  With
// m d = 2^p + e, 0 <= e < d, q is too large by r e / (d 2^p) < 1 / d: not enough to reach the next integer.
struct Divisor {
  unsigned m, shift;
  __host__ static Divisor of(int64_t d) {
    unsigned p = 31;
    while ((INT64_C(1) << (p - 31)) < d) ++p;
    return {(unsigned)(((INT64_C(1) << p) + d - 1) / d), p};
  }
  __device__ __forceinline__ unsigned divide(unsigned r) const { return (unsigned)((unsigned long long)r * m >> shift); }
};

// The scale of 4-bit codes that a byte stands for; 255 makes an infinity, which the conversions take for NaN.
__device__ __forceinline__ float scale_of_byte(unsigned b) { return __builtin_bit_cast(float, b << 23); }

// Largest magnitude of T that 4-bit codes have a value for: 6 times a power of two, and finite.
template <typename T>
constexpr float kMostF4 = std::is_same<T, Bf16>::value ? 0x1.8p127f : 49152.0f;
constexpr unsigned kLeastF4 = 27;  // byte of 2^-100, the least scale of 4-bit codes

// Eight elements f of a row, from element d on, as they come out of or go into T; a group of L lanes has the row, lanes with d >= dim
// nothing of it (but they call).
template <typename T, int CODES, int L>
__device__ __forceinline__ void put_elements(const CacheView &c, int which, long long slot, int h, int d, float (&f)[8]) {
  const long long page = slot >> c.page_log2, in = slot & ((1 << c.page_log2) - 1);
  const long long to = page * c.stride[0] + h * c.stride[1] + in * c.stride[2] + d;
  const long long scale_to = page * c.scale_stride[0] + h * c.scale_stride[1] + in * c.scale_stride[2];
  if constexpr (CODES == kNoCodes) {
    if (d < c.dim) *(vec8<T> *)((typename T::elem *)c.data[which] + to) = narrow<T>(f);
  } else if constexpr (CODES == kF8) {
    unsigned top = 0;  // of the finite and infinite elements: a NaN keeps its place and leaves its neighbours alone
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(f[i]) > kInfBits ? 0u : abs_bits(f[i]));
    const float amax = __builtin_bit_cast(float, group_max<L>(top));
    const float scale = amax / 448.0f;
    if (scale > 0.0f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] / scale;
    }
    if (d < c.dim) *(v2i *)(c.data[which] + to) = narrow_f8(f);
    if (d == 0) ((float *)c.scale[which])[scale_to] = scale;
  } else {
    // 32 elements are four lanes.  With 1.m * 2^e the largest magnitude, 6 * 2^(e - 2) holds it up to m = 0.5, 6 * 2^(e - 1) beyond.
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(f[i]));
    top = group_max<4>(top);
    const bool lost = top >= kInfBits;
    top = min(top, __builtin_bit_cast(unsigned, kMostF4<T>));
    const int exponent = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u);
    const unsigned byte = lost ? 255u : (unsigned)max(exponent, (int)kLeastF4);
    const float scale = scale_of_byte(lost ? kLeastF4 : byte);
    unsigned codes = 0;  // rounded to nearest even; beyond 6 they stay 6
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], scale, 3);
    if (d < c.dim) {
      *(unsigned *)(c.data[which] + to / 2) = codes;
      if (d % 32 == 0) ((unsigned char *)c.scale[which])[scale_to + d / 32] = (unsigned char)byte;
    }
  }
}

// Eight 4-bit codes as floats.
__device__ __forceinline__ void widen_f4(unsigned x, float scale, float *f) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 1),
           c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, scale, 3);
  f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1], f[4] = c[0], f[5] = c[1], f[6] = e[0], f[7] = e[1];
}

int check_cache(const char *what, const lapis_hip_kv_cache *cache);

}  // namespace lapis
