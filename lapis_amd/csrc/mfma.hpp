// Matrix instructions of the attention kernels, their operand layouts and the LDS tiles that feed them.
//
// 32x32x16 (A 32 x 16, B 16 x 32): lane l holds A[l & 31][8 (l >> 5) + j] and B[8 (l >> 5) + j][l & 31], j < 8, and of
// the result element r row 8 (r / 4) + 4 (l >> 5) + r % 4, column l & 31.
// 16x16x32 (A 16 x 32, B 32 x 16): lane l holds A[l & 15][8 (l >> 4) + j], B[8 (l >> 4) + j][l & 15] and of the result
// element r row 4 (l >> 4) + r, column l & 15.
//
// A product's result (say scores, keys x queries) becomes the next one's operand without leaving its lanes: the order of the
// contracted index is free as long as both operands keep it, so the other operand is read in the order in which the
// result's rows lie in the registers (rows_in_order below).
#pragma once
#include "attn.hpp"

namespace lapis {

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma32(vec8<Bf16> a, vec8<Bf16> b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mfma32(vec8<F16> a, vec8<F16> b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma16(vec8<Bf16> a, vec8<Bf16> b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma16(vec8<F16> a, vec8<F16> b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// x of the other half of the wavefront joined with one's own (lanes l and l ^ 32), without LDS
__device__ __forceinline__ float halves_max(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  const unsigned lo = p[0], hi = p[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  const unsigned lo = p[0], hi = p[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

__device__ __forceinline__ float rows_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  const unsigned a = p[0], b = p[1];
  return halves_max(fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  const unsigned a = p[0], b = p[1];
  return halves_sum(__builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
}

// Tiles of rows of DP 16-bit elements in LDS, the 16-byte pieces of a row in an order of its own, so that two ways of reading
// meet 64 different banks: 16 lanes that take the same piece of 16 neighbouring rows (an operand whose lanes are rows; the
// turn is another one for each of the rows that would share banks), and 32 lanes that take the same 64 bytes of four
// neighbouring rows (a transposing read; the turns of four rows differ in the bits that number 64 bytes).
template <int DP>
__device__ __forceinline__ int turn(int row) {
  return DP >= 128 ? (row & 3) << 2 | ((row >> 2) & 3) : ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
}
// A tile that is only read by columns takes the part of it that serves that: rows eight apart have the same order then, one
// address register fewer for each 32 columns (the forward kernel at dim 128 has none to spare: it keeps three in memory, outside its loop).
template <int DP>
__device__ __forceinline__ int column_turn(int row) {
  return DP >= 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
}
template <int DP, bool COLUMNS = false>
__device__ __forceinline__ int place_of(int row, int piece) {
  return row * DP + ((piece ^ (COLUMNS ? column_turn<DP>(row) : turn<DP>(row))) * 8);
}

// The same for transposing reads of 16 columns, 32 lanes meeting the same 32 bytes of eight neighbouring rows.
template <int DP>
__device__ __forceinline__ int turn16(int row) {
  return DP >= 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1;
}

// Transposing read: of the four rows and 16 columns that a group of 16 lanes points at (lane i: row i / 4, columns
// 4 (i % 4) ..), lane i gets column i of the four rows.
template <typename T>
__device__ __forceinline__ vec4<T> read_columns(const typename T::elem *p) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(vec4<T>, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p));
}

template <typename T>
__device__ __forceinline__ vec8<T> join(vec4<T> a, vec4<T> b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Operand of 32x32x16 whose lanes are columns d0 .. d0 + 31 of a tile and whose contracted index is its rows r0 .. r0 + 15
// in the order of a 32x32 result: element j of half h is row 8 (j / 4) + 4 h + j % 4.
template <typename T, int DP, bool COLUMNS = false>
__device__ __forceinline__ vec8<T> columns_in_order(const typename T::elem *tile, int r0, int d0, int lane) {
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), d = d0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const typename T::elem *p = tile + r0 * DP;
  return join<T>(read_columns<T>(p + place_of<DP, COLUMNS>(row, d >> 3) + (d & 7)), read_columns<T>(p + place_of<DP, COLUMNS>(row + 8, d >> 3) + (d & 7)));
}

// 16 bytes a lane from global memory straight into LDS, lane i's at `to` + 16 i: no registers between, so a tile can be on
// its way while the one before is computed.  Written as an instruction because the compiler, which cannot tell the buffers
// apart, would wait for it before the next LDS read; nobody may read the bytes before lds_loads_done() and a barrier.
__device__ __forceinline__ void load_to_lds(const void *from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
__device__ __forceinline__ void load_word_to_lds(const void *from, unsigned to) {  // 4 bytes a lane
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory");
}
// the same from `offset` bytes behind an address that all lanes share
__device__ __forceinline__ void load_to_lds(const void *from, unsigned offset, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from) : "memory");
}
__device__ __forceinline__ void load_word_to_lds(const void *from, unsigned offset, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(from) : "memory");
}
// the same to a place MORE bytes behind `to`
template <unsigned MORE>
__device__ __forceinline__ void load_to_lds_behind(const void *from, unsigned offset, unsigned to) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from), "n"(MORE) : "memory", "scc");
}
// all but the last N loads of this wavefront
template <int N = 0>
__device__ __forceinline__ void lds_loads_done() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <typename E>
__device__ __forceinline__ unsigned lds_address(const E *p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) E *)p;
}

// Any element that is infinite or NaN?  (An exponent of all ones, two elements a word: one more than that reaches the sign's bit.)
template <typename T>
__device__ __forceinline__ bool not_finite(vec8<T> x) {
  const unsigned mask = std::is_same<T, Bf16>::value ? 0x7f807f80u : 0x7c007c00u, one = std::is_same<T, Bf16>::value ? 0x00800080u : 0x04000400u;
  const v4u w = __builtin_bit_cast(v4u, x);
  return ((((w[0] & mask) + one) | ((w[1] & mask) + one) | ((w[2] & mask) + one) | ((w[3] & mask) + one)) & 0x80008000u) != 0;
}
template <typename T>
__device__ __forceinline__ vec8<T> finite_only(vec8<T> x) {
  const unsigned mask = std::is_same<T, Bf16>::value ? 0x7f80u : 0x7c00u;
  u16x8 b = __builtin_bit_cast(u16x8, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = (b[i] & mask) == mask ? 0 : b[i];
  return __builtin_bit_cast(vec8<T>, b);
}

}  // namespace lapis
