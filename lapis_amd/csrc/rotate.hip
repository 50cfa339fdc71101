// Rows turned by their positions, and on their way into a paged cache.
//
// Pair (x, y) of a row becomes (x cos - y sin, x sin + y cos) of an angle that is one for all heads of a token.  Bound by memory: 16384 tokens of 32 heads,
// dim 128, bf16, three axes, in 58 us (4.6 TB/s read and written, where a large copy reaches 4.7); a prompt of 32768 tokens, 32 heads of queries and 8 of keys and
// values, into 4-bit codes in 142 us (4.9 TB/s; 193 with divisions and with slots asked for after the angles, 158 with every lane working out its
// own row: vector instructions in 93 % of the cycles).  48 tokens into 8-bit codes take 4 us, the launch.
#include "kvcache.hpp"

namespace lapis {
namespace {

enum { kQuery = 0, kKey = 1, kValue = 2 };

struct TurnArgs {
  const char *x[3];  // queries, keys, values
  char *out;         // of queries
  long long x_stride[3][3], out_stride[3];
  int heads, all_heads;  // of queries; with keys and values
  int tokens, dim, axes, pairs;
  Divisor by_heads, by_tokens;  // all_heads, tokens
  long long rows;  // tokens of all batch entries times all heads
  bool neighbours;
  double sign;
  const int *positions;
  long long position_stride[3];
  const double *frequencies;
  const int *slots;
  CacheView cache;
};

// Where a row lies: its token (of all batch entries), batch entry, what it is, and which head.
struct Row {
  unsigned token, b, t, head;
  int kind;
  // Of the row `more` heads further.  (Selects of values: an index would be a load before the load.)
  __device__ __forceinline__ const char *data(const TurnArgs &a, unsigned more) const {
    const auto one_of = [&](auto q, auto k, auto v) { return kind == kQuery ? q : kind == kKey ? k : v; };
    const auto stride = [&](int i) { return one_of(a.x_stride[kQuery][i], a.x_stride[kKey][i], a.x_stride[kValue][i]); };
    return one_of(a.x[kQuery], a.x[kKey], a.x[kValue]) + 2 * (b * stride(0) + t * stride(1) + head * stride(2)) + 2 * (more * stride(2));
  }
};
__device__ __forceinline__ Row row_of(const TurnArgs &a, unsigned r) {
  Row x;
  x.token = a.by_heads.divide(r);
  x.head = r - x.token * a.all_heads;
  x.b = a.by_tokens.divide(x.token);
  x.t = x.token - x.b * a.tokens;
  x.kind = kQuery;
  if (x.head >= (unsigned)a.heads) {
    x.head -= a.heads;
    x.kind = kKey;
    if (x.head >= (unsigned)a.cache.heads) x.head -= a.cache.heads, x.kind = kValue;
  }
  return x;
}

// A row belongs to a group of L lanes, eight elements each, as where rows are stored without being turned; a workgroup has 256 / L * N of them, heads
// of a token side by side.  Cosines and sines are one for all heads of a token: they are computed once a workgroup, in 64 bits
// (positions of a million leave 32 bits no fraction), while the first rows are on their way, and read from LDS.  A lane reads the other
// elements of its pairs from memory a second time (out of L1): the row may be written over, but by this wavefront and after it.
// TOGETHER: the 64 / L rows that a wavefront has at a time are neighbouring heads of one token and of one kind, so that which rows they are and where
// they lie is worked out once for the wavefront, in scalar registers.
template <typename T, int CODES, int L, int N, bool TOGETHER>
__global__ __launch_bounds__(256) void turn_kernel(TurnArgs a) {
  typedef typename T::elem elem;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const long long block_row = (long long)linear_block() * (256 / L * N);
  if (block_row >= a.rows) return;
  const int d = (threadIdx.x % L) * 8, pairs = a.pairs;
  const unsigned last_row = (unsigned)(a.rows - 1), row0 = (unsigned)block_row + threadIdx.x / L;
  const bool inside = d < a.dim, whole = !a.neighbours && pairs % 8 == 0;  // whole: the other elements are eight neighbours too
  const int other = d < pairs ? d + pairs : d - pairs;
  const unsigned more = TOGETHER ? threadIdx.x % 64 / L : 0, wave_row = __builtin_amdgcn_readfirstlane(row0);
  const auto my_row = [&](int i) {
    if constexpr (TOGETHER) return row_of(a, min(wave_row + i * (256 / L), last_row + 1 - 64 / L));
    else return row_of(a, min(row0 + i * (256 / L), last_row));
  };
  vec8<T> x[N], y[N];
  int slots[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Row r = my_row(i);
    const elem *p = (const elem *)r.data(a, more);
    x[i] = y[i] = vec8<T>{};
    slots[i] = r.kind == kQuery ? -1 : a.slots[r.token];
    if (inside) {
      x[i] = *(const vec8<T> *)(p + d);
      if (whole && d < 2 * pairs && r.kind != kValue) y[i] = *(const vec8<T> *)(p + other);
    }
  }
  const unsigned t0 = a.by_heads.divide((unsigned)block_row), t1 = a.by_heads.divide(min((unsigned)block_row + (256 / L * N - 1), last_row));
  const int angles = (int)(t1 - t0 + 1) * pairs;
  float *cosines = lds, *sines = lds + angles;
  for (int i = threadIdx.x; i < angles; i += 256) {
    const unsigned tt = i / pairs, pair = i - tt * pairs, token = t0 + tt, b = a.by_tokens.divide(token), t = token - b * a.tokens;
    double angle = 0.0;
    for (int x = 0; x < a.axes; ++x)
      angle += (double)a.positions[x * a.position_stride[0] + b * a.position_stride[1] + t * a.position_stride[2]] * a.frequencies[x * pairs + pair];
    double s, c;
    sincospi(angle * 0.3183098861837906715, &s, &c);
    cosines[i] = (float)c;
    sines[i] = (float)(s * a.sign);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((TOGETHER ? wave_row : row0) + i * (256 / L) > last_row) return;
    const Row r = my_row(i);
    float f[8];
    widen<T>(x[i], f);
    const int at = (int)(r.token - t0) * pairs;
    if (inside && d < 2 * pairs && r.kind != kValue) {
      if (whole) {
        float g[8];
        widen<T>(y[i], g);
        const v4f *c = (const v4f *)(cosines + at + (d < pairs ? d : d - pairs)), *s = (const v4f *)(sines + at + (d < pairs ? d : d - pairs));
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] * c[j / 4][j % 4] + g[j] * (d < pairs ? -s[j / 4][j % 4] : s[j / 4][j % 4]);
      } else if (a.neighbours) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int pair = d / 2 + j;
          if (pair < pairs) {
            const float c = cosines[at + pair], s = sines[at + pair], lo = f[2 * j], hi = f[2 * j + 1];
            f[2 * j] = lo * c - hi * s;
            f[2 * j + 1] = hi * c + lo * s;
          }
        }
      } else {
        const elem *p = (const elem *)r.data(a, more);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = d + j;
          if (e < 2 * pairs) {
            const int pair = e < pairs ? e : e - pairs;
            const float c = cosines[at + pair], s = sines[at + pair], g = (float)p[e < pairs ? e + pairs : pair];
            f[j] = f[j] * c + g * (e < pairs ? -s : s);
          }
        }
      }
    }
    if (r.kind == kQuery) {
      if (inside) *(vec8<T> *)((elem *)a.out + r.b * a.out_stride[0] + r.t * a.out_stride[1] + r.head * a.out_stride[2] + more * a.out_stride[2] + d) = narrow<T>(f);
      continue;
    }
    const long long slot = slots[i];
    if (slot >= 0 && slot < a.cache.slots) put_elements<T, CODES, L>(a.cache, r.kind - kKey, slot, r.head + more, d, f);
  }
}

int read_rotation(const char *what, const lapis_hip_rotation &r, int64_t dim, bool some, TurnArgs *a) {
  LAPIS_REQUIRE(r.axes >= 0 && r.axes <= 8 && r.pairs >= 0 && 2ll * r.pairs <= dim, "%s: %d axes and %d pairs of rows of %lld elements", what, r.axes, r.pairs,
                (long long)dim);
  LAPIS_REQUIRE(!some || r.axes == 0 || r.pairs == 0 || (r.positions && r.frequencies), "%s: null positions or frequencies", what);
  a->axes = r.axes;
  a->pairs = r.pairs;
  a->neighbours = r.neighbours != 0;
  a->positions = r.positions;
  for (int i = 0; i < 3; ++i) a->position_stride[i] = r.position_stride[i];
  a->frequencies = r.frequencies;
  return LAPIS_HIP_OK;
}

int read_rows(const char *what, const lapis_hip_rows &r, const char **data, long long *stride) {
  LAPIS_REQUIRE(r.data && aligned16(r.data) && strides_of_8(r.stride, 3),
                "%s: rows that are null, not on a 16-byte boundary or with strides that are no multiples of 8", what);
  *data = static_cast<const char *>(r.data);
  for (int i = 0; i < 3; ++i) stride[i] = r.stride[i];
  return LAPIS_HIP_OK;
}

template <typename T, int CODES>
int launch_turn(TurnArgs a, hipStream_t st) {
  a.by_heads = Divisor::of(a.all_heads);
  a.by_tokens = Divisor::of(a.tokens);
  const auto go = [&](auto lanes, auto times, auto together) {
    constexpr int L = decltype(lanes)::value, N = decltype(times)::value, ROWS = 256 / L * N;
    constexpr bool TOGETHER = decltype(together)::value;
    const int64_t tokens = std::min<int64_t>(ROWS, (ROWS - 2) / a.all_heads + 2);  // that a workgroup has rows of, at most
    hipLaunchKernelGGL((turn_kernel<T, CODES, L, N, TOGETHER>), grid_of(ceil_div(a.rows, ROWS)), dim3(256), (size_t)(tokens * a.pairs * 8), st, a);
  };
  const auto with = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    // four rows a thread only where that leaves every compute unit its workgroups (the prompt above with its reading back: 183 us, with two rows 178, with
    // eight 184, and 193 where rows are each lane's own; the 16384 tokens 58, 63, 57 and 61)
    if (a.rows * L < 256 * 16 * device_cu_count()) go(lanes, std::integral_constant<int, 1>(), std::false_type());
    else if (a.heads % (64 / L) || a.cache.heads % (64 / L)) go(lanes, std::integral_constant<int, 4>(), std::false_type());
    else go(lanes, std::integral_constant<int, 4>(), std::true_type());
  };
  if (a.dim <= 64) with(std::integral_constant<int, 8>());
  else if (a.dim <= 128) with(std::integral_constant<int, 16>());
  else with(std::integral_constant<int, 32>());
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_rotate(int64_t batch, int64_t tokens, int64_t heads, int64_t dim, const lapis_hip_rotation *rotation, int inverse,
                                const lapis_hip_rows *x, const lapis_hip_rows *out, int dtype, lapis_hip_stream_t stream) {
  const char *what = "rotate";
  LAPIS_CHECK_INIT();
  LAPIS_REQUIRE(rotation && x && out, "%s: null arguments", what);
  LAPIS_REQUIRE(batch >= 0 && tokens >= 0 && heads >= 0, "%s: a negative size", what);
  LAPIS_REQUIRE(dim >= 8 && dim <= kMaxDim && dim % 8 == 0, "%s: rows of %lld elements (a multiple of 8 up to %d)", what, (long long)dim, kMaxDim);
  LAPIS_REQUIRE(is_16bit(dtype), "%s: rows of type %d", what, dtype);
  const bool some = batch && tokens && heads;
  TurnArgs a = {};
  int rc = read_rotation(what, *rotation, dim, some, &a);
  if (rc != LAPIS_HIP_OK || !some) return rc;
  LAPIS_REQUIRE(batch <= INT32_MAX && tokens <= INT32_MAX / batch && heads <= INT32_MAX / (batch * tokens), "%s: %lld x %lld tokens of %lld heads", what,
                (long long)batch, (long long)tokens, (long long)heads);
  const char *to;
  rc = read_rows(what, *x, &a.x[kQuery], a.x_stride[kQuery]);
  if (rc == LAPIS_HIP_OK) rc = read_rows(what, *out, &to, a.out_stride);
  if (rc != LAPIS_HIP_OK) return rc;
  a.out = const_cast<char *>(to);
  a.heads = a.all_heads = (int)heads;
  a.tokens = (int)tokens;
  a.dim = (int)dim;
  a.rows = batch * tokens * heads;
  a.sign = inverse ? -1.0 : 1.0;
  return dtype == LAPIS_HIP_BF16 ? launch_turn<Bf16, kNoCodes>(a, as_stream(stream)) : launch_turn<F16, kNoCodes>(a, as_stream(stream));
}

extern "C" int lapis_hip_kv_append(const lapis_hip_kv_cache *cache, const lapis_hip_append_args *p, lapis_hip_stream_t stream) {
  const char *what = "kv_append";
  int rc = check_cache(what, cache);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  LAPIS_REQUIRE(p->tokens >= 0 && p->q_heads >= 0, "%s: a negative size", what);
  LAPIS_REQUIRE(is_16bit(p->dtype) && (cache->dtype == p->dtype || codes_of(cache->dtype) != kNoCodes), "%s: rows of type %d and a cache of type %d", what,
                p->dtype, cache->dtype);
  TurnArgs a = {};
  rc = read_rotation(what, p->rotation, cache->dim, p->tokens > 0, &a);
  if (rc != LAPIS_HIP_OK || p->tokens == 0) return rc;
  LAPIS_REQUIRE(p->slots, "%s: null slots", what);
  const int64_t heads = 2ll * cache->heads;
  LAPIS_REQUIRE(p->q_heads <= INT32_MAX - heads && p->tokens <= INT32_MAX / (p->q_heads + heads), "%s: %lld tokens of %lld heads and %d of keys and values", what,
                (long long)p->tokens, (long long)p->q_heads, cache->heads);
  rc = read_rows(what, p->k, &a.x[kKey], a.x_stride[kKey]);
  if (rc == LAPIS_HIP_OK) rc = read_rows(what, p->v, &a.x[kValue], a.x_stride[kValue]);
  if (rc == LAPIS_HIP_OK && p->q_heads) {
    const char *to;
    rc = read_rows(what, p->q, &a.x[kQuery], a.x_stride[kQuery]);
    if (rc == LAPIS_HIP_OK) rc = read_rows(what, p->q_out, &to, a.out_stride);
    if (rc == LAPIS_HIP_OK) a.out = const_cast<char *>(to);
  }
  if (rc != LAPIS_HIP_OK) return rc;
  a.heads = (int)p->q_heads;
  a.all_heads = (int)(p->q_heads + heads);
  a.tokens = (int)p->tokens;
  a.dim = cache->dim;
  a.rows = p->tokens * a.all_heads;
  a.sign = 1.0;
  a.slots = p->slots;
  a.cache = view_of(cache);
  const hipStream_t st = as_stream(stream);
  const auto launch = [&](auto type) {
    typedef decltype(type) T;
    switch (codes_of(cache->dtype)) {
      case kF4: return launch_turn<T, kF4>(a, st);
      case kF8: return launch_turn<T, kF8>(a, st);
      default: return launch_turn<T, kNoCodes>(a, st);
    }
  };
  return p->dtype == LAPIS_HIP_BF16 ? launch(Bf16()) : launch(F16());
}
