// Keys and values into a cache of pages and back out of it, quantised to e4m3 with one scale per row on the way.
//
// A row of `dim` elements belongs to a group of lanes, eight elements each (one 16-byte load); the row's maximum is
// a DPP reduction over the group, so a row is read once and nothing is kept but registers.  Bound by memory: 32 768 tokens
// of 8 heads, dim 128, bf16 into e4m3 in 51.5 us (4.0 TB/s), 20 000 tokens, dim 96, back into f16 in 24.1 (3.9 TB/s), where a
// large copy reaches 4.75; four rows a thread on their way, loads first, where that leaves every compute unit its workgroups
// (one row a thread: 54 and 30).  48 tokens take 4.5 us, the call and the launch.
#include "attn.hpp"

namespace lapis {
namespace {

struct CacheView {
  char *data[2];
  float *scale[2];
  long long stride[3], scale_stride[3];
  long long slots;  // pages * page
  int heads, page_log2, dim;
};
struct RowsView {
  char *data[2];
  long long stride[2][2];  // token, head
};

CacheView view_of(const lapis_hip_kv_cache *c) {
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

// Group of L lanes per (token, head) and of N of them, 256 / L rows apart; blockIdx.z: keys or values.
template <typename T, bool F8, int L, int N>
__global__ __launch_bounds__(256) void kv_store_kernel(CacheView c, RowsView x, long long rows, const int *__restrict__ slots) {
  typedef typename T::elem elem;
  const long long row0 = (long long)linear_block() * (256 / L * N) + threadIdx.x / L;
  const int d = (threadIdx.x % L) * 8, which = blockIdx.z;
  vec8<T> read[N];
  int slot_of[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned row = (unsigned)min(row0 + i * (256 / L), rows - 1), t = row / (unsigned)c.heads, h = row - t * c.heads;
    slot_of[i] = slots[t];
    read[i] = vec8<T>{};
    if (d < c.dim) read[i] = load_stream((const vec8<T> *)((const elem *)x.data[which] + t * x.stride[which][0] + h * x.stride[which][1] + d));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long row = row0 + i * (256 / L);
    if (row >= rows) return;
    const int h = (int)((unsigned)row % (unsigned)c.heads);
    const long long slot = slot_of[i];
    if (slot < 0 || slot >= c.slots) continue;
    const long long page = slot >> c.page_log2, in = slot & ((1 << c.page_log2) - 1);
    const long long to = page * c.stride[0] + h * c.stride[1] + in * c.stride[2] + d;
    const vec8<T> e = read[i];
    if (!F8) {
      if (d < c.dim) *(vec8<T> *)((elem *)c.data[which] + to) = e;
      continue;
    }
    float f[8];
    widen<T>(e, f);
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
    if (d == 0) c.scale[which][page * c.scale_stride[0] + h * c.scale_stride[1] + in * c.scale_stride[2]] = scale;
  }
}

template <typename T, bool F8, int L, int N>
__global__ __launch_bounds__(256) void kv_load_kernel(CacheView c, RowsView x, long long rows, const int *__restrict__ slots) {
  typedef typename T::elem elem;
  typedef typename std::conditional<F8, v2i, v4i>::type raw;  // eight elements
  const long long row0 = (long long)linear_block() * (256 / L * N) + threadIdx.x / L;
  const int d = (threadIdx.x % L) * 8, which = blockIdx.z;
  if (d >= c.dim) return;
  raw read[N];
  float scale[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned row = (unsigned)min(row0 + i * (256 / L), rows - 1), t = row / (unsigned)c.heads, h = row - t * c.heads;
    const long long slot = slots[t];
    read[i] = raw{};
    scale[i] = 0.f;
    if (slot >= 0 && slot < c.slots) {
      const long long page = slot >> c.page_log2, in = slot & ((1 << c.page_log2) - 1);
      read[i] = load_stream((const raw *)(c.data[which] + (page * c.stride[0] + h * c.stride[1] + in * c.stride[2] + d) * (F8 ? 1 : 2)));
      if (F8) scale[i] = c.scale[which][page * c.scale_stride[0] + h * c.scale_stride[1] + in * c.scale_stride[2]];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long row = row0 + i * (256 / L);
    if (row >= rows) return;
    const unsigned t = (unsigned)row / (unsigned)c.heads, h = (unsigned)row - t * c.heads;
    vec8<T> e;
    if constexpr (F8) {
      float f[8];
      widen_f8(read[i], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * scale[i];
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
  LAPIS_REQUIRE(is_16bit(dtype) && (cache->dtype == dtype || cache->dtype == LAPIS_HIP_F8E4M3),
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
  const bool f8 = cache->dtype == LAPIS_HIP_F8E4M3, bf16 = dtype == LAPIS_HIP_BF16;
  const auto go = [&](auto lanes, auto times) {
    constexpr int L = decltype(lanes)::value, N = decltype(times)::value;
    const auto pick = [&](auto type) {
      typedef decltype(type) T;
      if (STORE) return f8 ? kv_store_kernel<T, true, L, N> : kv_store_kernel<T, false, L, N>;
      return f8 ? kv_load_kernel<T, true, L, N> : kv_load_kernel<T, false, L, N>;
    };
    dim3 grid = grid_of(ceil_div(rows * L, 256 * N));
    grid.z = 2;
    hipLaunchKernelGGL((bf16 ? pick(Bf16()) : pick(F16())), grid, dim3(256), 0, as_stream(stream), c, x, rows, slots);
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
  const bool f8 = c->dtype == LAPIS_HIP_F8E4M3;
  LAPIS_REQUIRE(f8 || is_16bit(c->dtype), "%s: a cache of type %d", what, c->dtype);
  if (c->pages == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(c->k && c->v && (!f8 || (c->k_scale && c->v_scale)), "%s: null cache buffers", what);
  const uintptr_t low = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v);
  LAPIS_REQUIRE((low & (f8 ? 7u : 15u)) == 0 && strides_of_8(c->stride, 3),
                "%s: cache buffers that are not on %d-byte boundaries or strides that are no multiples of 8", what, f8 ? 8 : 16);
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
