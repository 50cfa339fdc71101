// Keys and values into a cache of pages and back out of it, quantised on the way: to e4m3 with one scale per row, or to e2m1 with a power of two
// for each 32 elements.
//
// A row of `dim` elements belongs to a group of lanes, eight elements each (one 16-byte load); the row's maximum is
// a DPP reduction over the group, so a row is read once and nothing is kept but registers.  Bound by memory: 32 768 tokens
// of 8 heads, dim 128, bf16 into e4m3 in 50 us (4.1 TB/s), 20 000 tokens, dim 96, back into f16 in 22.1 (4.2 TB/s), where a
// large copy reaches 4.75; 32 768 tokens of 8 heads, dim 128, into 4-bit codes in 36 to 39 us and out of them in 41 (4.1 TB/s, most of it written); four rows a thread on their way, loads first, where that leaves every compute unit its workgroups
// (one row a thread: 54 and 30).  48 tokens take 4.5 us, the call and the launch.
#include "kvcache.hpp"

namespace lapis {
namespace {

// Group of L lanes per (token, head) and of N of them, 256 / L rows apart; blockIdx.z: keys or values.
template <typename T, int CODES, int L, int N>
__global__ __launch_bounds__(256) void kv_store_kernel(CacheView c, RowsView x, long long rows, Divisor by_heads, const int *__restrict__ slots) {
  typedef typename T::elem elem;
  const long long row0 = (long long)linear_block() * (256 / L * N) + threadIdx.x / L;
  const int d = (threadIdx.x % L) * 8, which = blockIdx.z;
  vec8<T> read[N];
  int slot_of[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned row = (unsigned)min(row0 + i * (256 / L), rows - 1), t = by_heads.divide(row), h = row - t * c.heads;
    slot_of[i] = slots[t];
    read[i] = vec8<T>{};
    if (d < c.dim) read[i] = load_stream((const vec8<T> *)((const elem *)x.data[which] + t * x.stride[which][0] + h * x.stride[which][1] + d));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long row = row0 + i * (256 / L);
    if (row >= rows) return;
    const int h = (int)((unsigned)row - by_heads.divide((unsigned)row) * c.heads);
    const long long slot = slot_of[i];
    if (slot < 0 || slot >= c.slots) continue;
    if constexpr (CODES == kNoCodes) {
      const long long page = slot >> c.page_log2, in = slot & ((1 << c.page_log2) - 1);
      if (d < c.dim) *(vec8<T> *)((elem *)c.data[which] + page * c.stride[0] + h * c.stride[1] + in * c.stride[2] + d) = read[i];
    } else {
      float f[8];
      widen<T>(read[i], f);
      put_elements<T, CODES, L>(c, which, slot, h, d, f);
    }
  }
}

template <typename T, int CODES, int L, int N>
__global__ __launch_bounds__(256) void kv_load_kernel(CacheView c, RowsView x, long long rows, Divisor by_heads, const int *__restrict__ slots) {
  typedef typename T::elem elem;
  typedef typename std::conditional<CODES == kF8, v2i, typename std::conditional<CODES == kF4, unsigned, v4i>::type>::type raw;  // eight elements
  const long long row0 = (long long)linear_block() * (256 / L * N) + threadIdx.x / L;
  const int d = (threadIdx.x % L) * 8, which = blockIdx.z;
  if (d >= c.dim) return;
  raw read[N];
  float scale[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned row = (unsigned)min(row0 + i * (256 / L), rows - 1), t = by_heads.divide(row), h = row - t * c.heads;
    const long long slot = slots[t];
    read[i] = raw{};
    scale[i] = 0.f;
    if (slot >= 0 && slot < c.slots) {
      const long long page = slot >> c.page_log2, in = slot & ((1 << c.page_log2) - 1);
      const long long at = page * c.stride[0] + h * c.stride[1] + in * c.stride[2] + d;
      read[i] = load_stream((const raw *)(c.data[which] + (CODES == kF4 ? at / 2 : CODES == kF8 ? at : at * 2)));
      const long long scale_at = page * c.scale_stride[0] + h * c.scale_stride[1] + in * c.scale_stride[2];
      if (CODES == kF8) scale[i] = ((const float *)c.scale[which])[scale_at];
      if (CODES == kF4) scale[i] = scale_of_byte(((const unsigned char *)c.scale[which])[scale_at + d / 32]);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long row = row0 + i * (256 / L);
    if (row >= rows) return;
    const unsigned t = by_heads.divide((unsigned)row), h = (unsigned)row - t * c.heads;
    vec8<T> e;
    if constexpr (CODES != kNoCodes) {
      float f[8];
      if constexpr (CODES == kF4) {
        widen_f4(read[i], scale[i], f);
      } else {
        widen_f8(read[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] * scale[i];
      }
      e = narrow<T>(f);
    } else {
      e = __builtin_bit_cast(vec8<T>, read[i]);
    }
    *(vec8<T> *)((elem *)x.data[which] + t * x.stride[which][0] + h * x.stride[which][1] + d) = e;
  }
}

template <bool STORE>
int kv_move(const char *what, const lapis_hip_kv_cache *cache, int64_t tokens, const lapis_hip_rows *k, const lapis_hip_rows *v,
            int dtype, const int32_t *slots, lapis_hip_stream_t stream) {
  const int rc = check_cache(what, cache);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(k && v && tokens >= 0, "%s: null rows or a negative number of tokens", what);
  LAPIS_REQUIRE(is_16bit(dtype) && (cache->dtype == dtype || codes_of(cache->dtype) != kNoCodes),
                "%s: rows of type %d and a cache of type %d", what, dtype, cache->dtype);
  if (tokens == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(slots, "%s: null slots", what);
  LAPIS_REQUIRE(tokens <= INT32_MAX / cache->heads, "%s: %lld tokens of %d heads", what, (long long)tokens, cache->heads);
  const long long rows = tokens * cache->heads;
  for (const lapis_hip_rows *r : {k, v})
    LAPIS_REQUIRE(r->data && aligned16(r->data) && strides_of_8(r->stride + 1, 2),
                  "%s: rows that are null, not on a 16-byte boundary or with strides that are no multiples of 8", what);
  const CacheView c = view_of(cache);
  RowsView x = {{static_cast<char *>(k->data), static_cast<char *>(v->data)}, {{k->stride[1], k->stride[2]}, {v->stride[1], v->stride[2]}}};
  const Codes codes = codes_of(cache->dtype);
  const bool bf16 = dtype == LAPIS_HIP_BF16;
  const auto go = [&](auto lanes, auto times) {
    constexpr int L = decltype(lanes)::value, N = decltype(times)::value;
    const auto pick = [&](auto type) {
      typedef decltype(type) T;
      if (STORE) return codes == kF4 ? kv_store_kernel<T, kF4, L, N> : codes == kF8 ? kv_store_kernel<T, kF8, L, N> : kv_store_kernel<T, kNoCodes, L, N>;
      return codes == kF4 ? kv_load_kernel<T, kF4, L, N> : codes == kF8 ? kv_load_kernel<T, kF8, L, N> : kv_load_kernel<T, kNoCodes, L, N>;
    };
    dim3 grid = grid_of(ceil_div(rows * L, 256 * N));
    grid.z = 2;
    hipLaunchKernelGGL((bf16 ? pick(Bf16()) : pick(F16())), grid, dim3(256), 0, as_stream(stream), c, x, rows, Divisor::of(c.heads), slots);
  };
  const auto with = [&](auto lanes) {
    // four rows a thread only where that leaves every compute unit its workgroups
    if (rows * decltype(lanes)::value >= 256 * 16 * device_cu_count()) go(lanes, std::integral_constant<int, 4>());
    else go(lanes, std::integral_constant<int, 1>());
  };
  if (cache->dim <= 64) with(std::integral_constant<int, 8>());
  else if (cache->dim <= 128) with(std::integral_constant<int, 16>());
  else with(std::integral_constant<int, 32>());
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

}  // namespace

int check_cache(const char *what, const lapis_hip_kv_cache *c) {
  LAPIS_CHECK_INIT();
  LAPIS_REQUIRE(c, "%s: null cache", what);
  LAPIS_REQUIRE(c->heads > 0 && c->pages >= 0, "%s: a cache of %lld pages and %d heads", what, (long long)c->pages, c->heads);
  LAPIS_REQUIRE(c->page >= 1 && c->page <= 1024 && (c->page & (c->page - 1)) == 0, "%s: pages of %d slots (a power of two up to 1024)", what, c->page);
  LAPIS_REQUIRE(c->pages <= INT32_MAX / c->page, "%s: %lld pages of %d slots: slots are numbered with 31 bits", what, (long long)c->pages, c->page);
  LAPIS_REQUIRE(c->dim >= 8 && c->dim <= kMaxDim && c->dim % 8 == 0, "%s: rows of %d elements (a multiple of 8 up to %d)", what, c->dim, kMaxDim);
  const Codes codes = codes_of(c->dtype);
  LAPIS_REQUIRE(codes != kNoCodes || is_16bit(c->dtype), "%s: a cache of type %d", what, c->dtype);
  LAPIS_REQUIRE(codes != kF4 || c->dim % 32 == 0, "%s: rows of %d elements in 4 bits (a multiple of 32)", what, c->dim);
  if (c->pages == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(c->k && c->v && (codes == kNoCodes || (c->k_scale && c->v_scale)), "%s: null cache buffers", what);
  const uintptr_t low = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v);
  const int boundary = codes == kF8 ? 8 : 16, strides = codes == kF4 ? 32 : 8;
  for (int i = 0; i < 3; ++i)
    LAPIS_REQUIRE((low & (boundary - 1u)) == 0 && c->stride[i] % strides == 0,
                  "%s: cache buffers that are not on %d-byte boundaries or strides that are no multiples of %d", what, boundary, strides);
  return LAPIS_HIP_OK;
}

}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_kv_store(const lapis_hip_kv_cache *cache, int64_t tokens, const lapis_hip_rows *k, const lapis_hip_rows *v,
                                  int dtype, const int32_t *slots, lapis_hip_stream_t stream) {
  return kv_move<true>("kv_store", cache, tokens, k, v, dtype, slots, stream);
}

extern "C" int lapis_hip_kv_load(const lapis_hip_kv_cache *cache, int64_t tokens, const int32_t *slots, const lapis_hip_rows *k,
                                 const lapis_hip_rows *v, int dtype, lapis_hip_stream_t stream) {
  return kv_move<false>("kv_load", cache, tokens, k, v, dtype, slots, stream);
}
