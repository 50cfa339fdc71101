// Which blocks of keys a block of queries attends to: 8-bit means of blocks, and the best-scoring ones as a CSR structure.
//
// A score is a product of whole numbers times the block's scale.  |code| <= 127, so a dot product of up to 1024 codes
// stays below 2^24 and is exact in fp32: the selection is the same whatever the order of summation.
#include "attn.hpp"

namespace lapis {
namespace {

// ---- pooling --------------------------------------------------------------------------------------------------

struct PoolArgs {
  const char *x;
  long long stride[3];
  long long tokens, blocks, lists_blocks;  // blocks of a list, blocks of all lists
  long long block;
  int groups, group, dim;
  signed char *codes;
  float *scales;
};

// A wavefront takes 64 / (L * PARTS) blocks: groups of L lanes hold a row (8 elements each), PARTS of them share a block's
// rows.  The rows of a block are summed in fp32, part by part, then over the parts.
template <typename T, int L, int PARTS>
__global__ __launch_bounds__(256) void block_pool_kernel(PoolArgs a) {
  const long long thread = (long long)linear_block() * 256 + threadIdx.x;
  const long long at = thread / (L * PARTS);
  const int part = (int)(thread / L) % PARTS, d = (int)(thread % L) * 8;
  const bool live = at < a.lists_blocks;
  const long long list = live ? at / a.blocks : 0, j = live ? at - list * a.blocks : 0;
  const long long b = list / a.groups;
  const int h0 = (int)(list - b * a.groups) * a.group;
  const long long t0 = j * a.block;
  const long long held = live ? min(a.block, a.tokens - t0) : 0;
  float sum[8] = {};
  if (d < a.dim) {
    const typename T::elem *x = (const typename T::elem *)a.x + b * a.stride[0] + d;
    const long long n = held * a.group;
    // row i of the block is token i / group, head i % group
    long long t = part / a.group;
    int h = part % a.group;
    for (long long i = part; i < n; i += PARTS) {
      float f[8];
      widen<T>(*(const vec8<T> *)(x + (t0 + t) * a.stride[1] + (h0 + h) * a.stride[2]), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += f[e];
      h += PARTS;
      while (h >= a.group) {
        h -= a.group;
        ++t;
      }
    }
  }
  if (PARTS > 1) {
#pragma unroll
    for (int o = L; o < L * PARTS; o *= 2)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], o, 64);
  }
  const float count = (float)(held * a.group);
  unsigned top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    sum[e] = sum[e] / count;
    if (d < a.dim) top = max(top, abs_bits(sum[e]));
  }
  top = group_max<L>(top);
  const bool finite = top < kInfBits;
  const float scale = finite ? __builtin_bit_cast(float, top) / 127.0f : __builtin_nanf("");
  unsigned packed[2] = {0, 0};
  if (finite && scale > 0.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = fminf(fmaxf(rintf(sum[e] / scale), -127.0f), 127.0f);
      packed[e / 4] |= ((unsigned)(int)q & 0xffu) << (8 * (e % 4));
    }
  }
  if (!live || part != 0 || d >= a.dim) return;
  *(v2u *)(a.codes + at * a.dim + d) = v2u{packed[0], packed[1]};
  if (d == 0) a.scales[at] = scale;
}

// ---- selection ------------------------------------------------------------------------------------------------

struct SelectArgs {
  long long batch, heads, rows;  // rows of a list
  long long queries, keys, block_m, block_n, columns, count, sink, local;
  int causal, dim;
  const signed char *q, *k;
  const float *scales;
  long long k_stride[3], scale_stride[3];
  const int *table, *blocks;
  long long table_width, pages;
  int *pos, *crd;
  long long list_entries;  // of one list, where every list has the same
};

__host__ __device__ inline long long floor_div(long long a, long long b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

// sum over i < n of floor((a i + b) / m), all non-negative, by the steps of Euclid's algorithm
__host__ __device__ inline long long floor_sum(long long n, long long m, long long a, long long b) {
  long long total = 0;
  while (n > 0) {
    if (a >= m) total += (n - 1) * n / 2 * (a / m), a %= m;
    if (b >= m) total += n * (b / m), b %= m;
    const long long top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const long long t = m;
    m = a;
    a = t;
  }
  return total;
}

// Blocks that row r may see (causal or all of `columns`).
__host__ __device__ inline long long blocks_seen(const SelectArgs &a, long long r) {
  if (!a.causal) return a.columns;
  const long long end = (r + 1) * a.block_m, last = (end < a.queries ? end : a.queries) - 1;
  const long long n = floor_div(last + a.keys - a.queries, a.block_n) + 1;
  return n < 0 ? 0 : n < a.columns ? n : a.columns;
}

// Entries of the rows before row r of a list: min(count, seen) grows with r in three stretches (none, floor((block_m i +
// c) / block_n), all `cap`), so no row needs another one's answer.
__host__ __device__ inline long long entries_before(const SelectArgs &a, long long r) {
  const long long cap = a.count < a.columns ? a.count : a.columns;
  if (!a.causal) return r * cap;
  if (r <= 0) return 0;
  const long long before = r < a.rows ? r : a.rows - 1;  // the last row's end is cut: it is added by itself
  const long long c = a.block_m - 1 + a.keys - a.queries + a.block_n;
  long long i0 = -floor_div(c - a.block_n, a.block_m), i1 = -floor_div(c - cap * a.block_n, a.block_m);
  i0 = i0 < 0 ? 0 : i0;
  i1 = i1 < i0 ? i0 : i1;
  const long long stop = before < i1 ? before : i1;
  long long total = stop > i0 ? floor_sum(stop - i0, a.block_n, a.block_m, a.block_m * i0 + c) : 0;
  if (before > i1) total += (before - i1) * cap;
  if (r == a.rows) {
    const long long seen = blocks_seen(a, r - 1);
    total += seen < cap ? seen : cap;
  }
  return total;
}

// Scores as unsigned numbers in the same order, NaN first.
__device__ __forceinline__ unsigned sortable(float x) {
  if (x != x) return 0u;
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);  // -0 becomes 0
  return b >> 31 ? ~b : b | 0x80000000u;
}

// One wavefront per row; `key(j)` gives block j's score.  A candidate's bits are found from the top: the largest
// threshold that still leaves `need` blocks at or above it.
template <typename Key>
__device__ __forceinline__ void take_best(const SelectArgs &a, long long seen, int *out, int lane, Key key,
                                          const int *__restrict__ table) {
  const long long need = seen < a.count ? seen : a.count;
  unsigned threshold = 0;
  if (need < seen) {
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned candidate = threshold | (1u << bit);
      int n = 0;
      for (long long j = lane; j < seen; j += 64) n += key(j) >= candidate;
      n = group_sum<64>(n);
      if (n >= need) threshold = candidate;
    }
  }
  long long above = 0;
  if (need < seen) {
    int n = 0;
    for (long long j = lane; j < seen; j += 64) n += key(j) > threshold;
    above = group_sum<64>(n);
  }
  long long equal_left = need - above, at = 0;
  for (long long j0 = 0; j0 < seen && at < need; j0 += 64) {
    const long long j = j0 + lane;
    bool take = j < seen;
    if (need < seen) {
      const unsigned k = take ? key(j) : 0u;
      const bool equal = take && k == threshold;
      const unsigned long long ties = __ballot(equal);
      const int before = __popcll(ties & ((1ull << lane) - 1));
      take = take && (k > threshold || (equal && before < equal_left));
      equal_left -= min((long long)__popcll(ties), equal_left);
    }
    const unsigned long long taken = __ballot(take);
    if (take) out[at + __popcll(taken & ((1ull << lane) - 1))] = table ? table[j] : (int)j;
    at += __popcll(taken);
  }
}

__device__ __forceinline__ float block_score(const SelectArgs &a, long long b, long long h, const signed char *q, long long j) {
  long long page = j;
  const signed char *k = a.k + h * a.k_stride[1];
  const float *s = a.scales + h * a.scale_stride[1];
  if (a.table) {
    page = a.table[b * a.table_width + j];
    if (page < 0 || page >= a.pages) return __builtin_nanf("");
  } else {
    k += b * a.k_stride[0];
    s += b * a.scale_stride[0];
  }
  k += page * a.k_stride[2];
  int dot = 0;
  for (int d = 0; d < a.dim; d += 8) {
    const v2i x = *(const v2i *)(q + d), y = *(const v2i *)(k + d);
    dot = __builtin_amdgcn_sdot4(x[0], y[0], dot, false);
    dot = __builtin_amdgcn_sdot4(x[1], y[1], dot, false);
  }
  return (float)dot * s[page * a.scale_stride[2]];
}

__global__ __launch_bounds__(64) void block_select_kernel(SelectArgs a, unsigned *scores) {
  const long long row = linear_block();
  const int lane = threadIdx.x;
  const long long lists = a.batch * a.heads;
  if (row >= lists * a.rows) return;
  const long long list = row / a.rows, r = row - list * a.rows, b = list / a.heads, h = list - b * a.heads;
  long long seen, first;
  if (a.blocks) {
    long long before = 0;
    for (long long i = lane; i < b; i += 64) {
      const long long n = max(0ll, min((long long)a.blocks[i], a.columns));
      before += min(n, a.count);
    }
    for (int o = 1; o < 64; o <<= 1) before += __shfl_xor(before, o, 64);
    seen = max(0ll, min((long long)a.blocks[b], a.columns));
    first = before * a.heads * a.rows + (h * a.rows + r) * min(seen, a.count);
  } else {
    seen = blocks_seen(a, r);
    first = list * a.list_entries + entries_before(a, r);
  }
  if (lane == 0) {
    a.pos[row] = (int)first;
    if (row == lists * a.rows - 1) a.pos[row + 1] = (int)(first + min(seen, a.count));
  }
  unsigned *mine = scores + row * a.columns;
  if (seen > a.count)
    for (long long j = lane; j < seen; j += 64)
      mine[j] = j < a.sink || j >= seen - a.local ? 0xffffffffu : sortable(block_score(a, b, h, a.q + row * a.dim, j));
  const int *table = a.table ? a.table + b * a.table_width : nullptr;
  take_best(a, seen, a.crd + first, lane, [&](long long j) { return mine[j]; }, table);
}

__global__ void empty_positions_kernel(int *pos) { pos[0] = 0; }

int read_select(const char *what, const lapis_hip_select_args *p, SelectArgs *a) {
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  LAPIS_REQUIRE(p->batch >= 0 && p->heads >= 0 && p->queries >= 0 && p->keys >= 0, "%s: a negative size", what);
  LAPIS_REQUIRE(p->block_m >= 1 && p->block_n >= 1, "%s: blocks of %lld queries and %lld keys", what, (long long)p->block_m, (long long)p->block_n);
  LAPIS_REQUIRE(p->queries <= INT32_MAX && p->keys <= INT32_MAX && p->block_m <= INT32_MAX && p->block_n <= INT32_MAX,
                "%s: sizes beyond 31 bits", what);
  LAPIS_REQUIRE(p->dim >= 8 && p->dim <= 1024 && p->dim % 8 == 0, "%s: codes of %lld elements (a multiple of 8 up to 1024)", what, (long long)p->dim);
  LAPIS_REQUIRE(p->count >= 1 && p->sink >= 0 && p->local >= 0 && p->sink + p->local <= p->count,
                "%s: %lld blocks a row, %lld first and %lld last ones among them", what, (long long)p->count, (long long)p->sink, (long long)p->local);
  LAPIS_REQUIRE(!p->causal || (!p->table && !p->blocks), "%s: causal rows over a table of pages", what);
  *a = {};
  a->batch = p->batch;
  a->heads = p->heads;
  a->queries = p->queries;
  a->keys = p->keys;
  a->block_m = p->block_m;
  a->block_n = p->block_n;
  a->rows = ceil_div(p->queries, p->block_m);
  a->columns = p->table ? p->table_width : ceil_div(p->keys, p->block_n);
  a->count = p->count;
  a->sink = p->sink;
  a->local = p->local;
  a->causal = p->causal;
  a->dim = (int)p->dim;
  a->q = p->q_codes;
  a->k = p->k_codes;
  a->scales = p->k_scales;
  for (int i = 0; i < 3; ++i) a->k_stride[i] = p->k_stride[i], a->scale_stride[i] = p->scale_stride[i];
  a->table = p->table;
  a->blocks = p->blocks;
  a->table_width = p->table_width;
  a->pages = p->pages;
  a->pos = p->pos;
  a->crd = p->crd;
  LAPIS_REQUIRE(a->columns >= 0 && a->columns <= INT32_MAX, "%s: %lld blocks", what, (long long)a->columns);
  a->list_entries = a->rows ? entries_before(*a, a->rows) : 0;
  const double lists = (double)p->batch * (double)p->heads;
  LAPIS_REQUIRE(lists * (double)a->rows < 2147483647.0 && lists * (double)a->list_entries < 2147483647.0,
                "%s: more rows or entries than 31 bits count", what);
  return LAPIS_HIP_OK;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_block_pool(int64_t batch, int64_t tokens, int64_t heads, int64_t groups, int64_t dim, int64_t block,
                                    const lapis_hip_rows *x, int dtype, int8_t *codes, float *scales, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  LAPIS_REQUIRE(x && batch >= 0 && tokens >= 0 && heads >= 0, "block_pool: null rows or a negative size");
  LAPIS_REQUIRE(groups >= 1 && heads % groups == 0 && groups <= INT32_MAX && heads <= INT32_MAX, "block_pool: %lld heads in %lld groups", (long long)heads, (long long)groups);
  LAPIS_REQUIRE(dim >= 8 && dim <= kMaxDim && dim % 8 == 0, "block_pool: rows of %lld elements (a multiple of 8 up to %d)", (long long)dim, kMaxDim);
  LAPIS_REQUIRE(block >= 1, "block_pool: blocks of %lld tokens", (long long)block);
  LAPIS_REQUIRE(is_16bit(dtype), "block_pool: rows of type %d", dtype);
  PoolArgs a = {static_cast<char *>(x->data), {x->stride[0], x->stride[1], x->stride[2]}, tokens, ceil_div(tokens, block),
                batch * groups * ceil_div(tokens, block), block, (int)groups, (int)(heads / groups), (int)dim, (signed char *)codes, scales};
  if (a.lists_blocks == 0 || heads == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(codes && scales && x->data, "block_pool: null operands");
  LAPIS_REQUIRE(aligned16(x->data) && strides_of_8(x->stride, 3) && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0,
                "block_pool: rows that are not on 16-byte boundaries, strides that are no multiples of 8, or codes that are not on an 8-byte boundary");
  LAPIS_REQUIRE(a.lists_blocks <= (INT64_C(1) << 33), "block_pool: %lld blocks", (long long)a.lists_blocks);
  const auto go = [&](auto lanes, auto parts) {
    constexpr int L = decltype(lanes)::value, P = decltype(parts)::value;
    const auto kernel = dtype == LAPIS_HIP_BF16 ? block_pool_kernel<Bf16, L, P> : block_pool_kernel<F16, L, P>;
    hipLaunchKernelGGL(kernel, grid_of(ceil_div(a.lists_blocks * L * P, 256)), dim3(256), 0, as_stream(stream), a);
  };
  // a wavefront per block, or where a block is a single row a group of lanes
  const bool one = block * a.group == 1;
  if (dim <= 64) one ? go(std::integral_constant<int, 8>(), std::integral_constant<int, 1>()) : go(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  else if (dim <= 128) one ? go(std::integral_constant<int, 16>(), std::integral_constant<int, 1>()) : go(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
  else one ? go(std::integral_constant<int, 32>(), std::integral_constant<int, 1>()) : go(std::integral_constant<int, 32>(), std::integral_constant<int, 2>());
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

extern "C" int lapis_hip_block_select_entries(const lapis_hip_select_args *args, int64_t *entries) {
  SelectArgs a;
  const int rc = read_select("block_select", args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(entries, "block_select: null result");
  *entries = a.batch * a.heads * a.list_entries;
  return LAPIS_HIP_OK;
}

extern "C" int lapis_hip_block_select_work(const lapis_hip_select_args *args, int64_t *bytes) {
  SelectArgs a;
  const int rc = read_select("block_select", args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "block_select: null result");
  *bytes = 4 * a.batch * a.heads * a.rows * a.columns;
  return LAPIS_HIP_OK;
}

extern "C" int lapis_hip_block_select(const lapis_hip_select_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  SelectArgs a;
  const int rc = read_select("block_select", args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  const long long rows = a.batch * a.heads * a.rows;
  LAPIS_REQUIRE(a.pos, "block_select: null positions");
  if (rows == 0 || a.columns == 0) {
    if (rows == 0) {
      hipLaunchKernelGGL(empty_positions_kernel, dim3(1), dim3(1), 0, as_stream(stream), a.pos);
      LAPIS_LAUNCH_CHECK();
      return LAPIS_HIP_OK;
    }
  } else {
    LAPIS_REQUIRE(a.q && a.k && a.scales && a.crd && args->work, "block_select: null operands");
    const uintptr_t low = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k);
    LAPIS_REQUIRE((low & 7u) == 0 && strides_of_8(args->k_stride, 3), "block_select: codes that are not on 8-byte boundaries or strides that are no multiples of 8");
  }
  hipLaunchKernelGGL(block_select_kernel, grid_of(rows), dim3(64), 0, as_stream(stream), a, static_cast<unsigned *>(args->work));
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}
