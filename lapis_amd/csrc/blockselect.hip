// Which blocks of keys a block of queries attends to: 8-bit means of blocks, and the best-scoring ones as a CSR structure.
//
// A score is a product of whole numbers times the block's scale.  |code| <= 127, so a dot product of up to 1024 codes
// stays below 2^24 and is exact in fp32: the selection is the same whatever the order of summation.
#include "attn.hpp"

namespace lapis {
namespace {

// 64-bit division takes a hundred instructions on the device; most operands here fit 32 bits.
__host__ __device__ inline long long quotient(long long a, long long b) {  // both non-negative
  return ((unsigned long long)(a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
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

// Bound by memory: 32 768 tokens of 8 heads, dim 128, bf16, blocks of 64: 12.5 us in a trace for 67 MB that the last-level
// cache partly holds.
// A wavefront takes 64 / (L * PARTS) blocks: groups of L lanes hold a row (8 elements each), PARTS of them share a block's
// rows.  The rows of a block are summed in fp32, part by part, then over the parts.
template <typename T, int L, int PARTS>
__global__ __launch_bounds__(256) void block_pool_kernel(PoolArgs a) {
  const long long thread = (long long)linear_block() * 256 + threadIdx.x;
  const long long at = thread / (L * PARTS);
  const int part = (int)(thread / L % PARTS), d = (int)(thread % L) * 8;
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
    // row i of the block is token i / group, head i % group; four rows on their way at a time
    const auto at_row = [&](long long i) {
      const long long t = a.group == 1 ? i : quotient(i, a.group);
      return x + (t0 + t) * a.stride[1] + (h0 + (int)(i - t * a.group)) * a.stride[2];
    };
    for (long long i = part; i < n; i += 4 * PARTS) {
      vec8<T> read[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) read[u] = i + u * PARTS < n ? load_stream((const vec8<T> *)at_row(i + u * PARTS)) : vec8<T>{};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float f[8];
        widen<T>(read[u], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += f[e];
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
  // entries_before()'s stretches, the same for all rows; step_rows > 0: block_n is a multiple of block_m, and then
  // floor((block_m i + c) / block_n) is floor((i + shift) / step_rows)
  long long first_row, full_row, shift, step_rows, steps_before;
};

__host__ __device__ inline long long floor_div(long long a, long long b) { return a >= 0 ? quotient(a, b) : -quotient(-a + b - 1, b); }

// sum over i < n of floor((a i + b) / m), all non-negative, by the steps of Euclid's algorithm
__host__ __device__ inline long long floor_sum(long long n, long long m, long long a, long long b) {
  long long total = 0;
  while (n > 0) {
    if (a >= m) {
      const long long q = quotient(a, m);
      total += (n - 1) * n / 2 * q;
      a -= q * m;
    }
    if (b >= m) {
      const long long q = quotient(b, m);
      total += n * q;
      b -= q * m;
    }
    const long long top = a * n + b;
    if (top < m) break;
    n = quotient(top, m);
    b = top - n * m;
    const long long t = m;
    m = a;
    a = t;
  }
  return total;
}

// Blocks that row r may see (causal or all of `columns`).  Queries and keys are counted with 31 bits.
__host__ __device__ inline long long blocks_seen(const SelectArgs &a, long long r) {
  if (!a.causal) return a.columns;
  const long long end = (r + 1) * a.block_m, last = (end < a.queries ? end : a.queries) - 1 + a.keys - a.queries;
  if (last < 0) return 0;
  const long long n = (unsigned)last / (unsigned)a.block_n + 1;
  return n < a.columns ? n : a.columns;
}

// Sum over x below y of floor(x / q).
__host__ __device__ inline long long stairs(long long y, long long q) {
  const long long k = quotient(y, q);
  return q * (k * (k - 1) / 2) + k * (y - k * q);
}

// Entries of the rows before row r of a list: min(count, seen) grows with r in three stretches (none, floor((block_m i +
// c) / block_n), all `cap`), so no row needs another one's answer.
__host__ __device__ inline long long entries_before(const SelectArgs &a, long long r) {
  const long long cap = a.count < a.columns ? a.count : a.columns;
  if (!a.causal) return r * cap;
  if (r <= 0) return 0;
  const long long before = r < a.rows ? r : a.rows - 1;  // the last row's end is cut: it is added by itself
  const long long stop = before < a.full_row ? before : a.full_row;
  long long total = 0;
  if (stop > a.first_row) {
    if (a.step_rows > 0) total = stairs(stop + a.shift, a.step_rows) - a.steps_before;
    else total = floor_sum(stop - a.first_row, a.block_n, a.block_m, a.block_m * (a.first_row + 1) - 1 + a.keys - a.queries + a.block_n);
  }
  if (before > a.full_row) total += (before - a.full_row) * cap;
  if (r == a.rows) {
    const long long seen = blocks_seen(a, r - 1);
    total += seen < cap ? seen : cap;
  }
  return total;
}

// The stretches: the first row that sees a block, and the first that sees `cap`.
inline void set_stretches(SelectArgs *a) {
  const long long cap = a->count < a->columns ? a->count : a->columns, c = a->block_m - 1 + a->keys - a->queries + a->block_n;
  a->first_row = -floor_div(c - a->block_n, a->block_m);
  a->full_row = -floor_div(c - cap * a->block_n, a->block_m);
  if (a->first_row < 0) a->first_row = 0;
  if (a->full_row < a->first_row) a->full_row = a->first_row;
  a->step_rows = a->block_n % a->block_m == 0 ? a->block_n / a->block_m : 0;
  a->shift = floor_div(c, a->block_m);
  // from first_row on every term is at least 1, so i + shift is not negative there
  if (a->step_rows > 0 && a->first_row + a->shift >= 0) a->steps_before = stairs(a->first_row + a->shift, a->step_rows);
  else a->step_rows = 0;
}

// Scores as unsigned numbers in the same order, NaN first.
__device__ __forceinline__ unsigned sortable_number(float x) {  // not NaN
  const int b = __builtin_bit_cast(int, x + 0.0f);  // -0 becomes 0
  return (unsigned)(b ^ (b >> 31 | (int)0x80000000));
}
__device__ __forceinline__ unsigned sortable(float x) { return x != x ? 0u : sortable_number(x); }

// What a row may see, and where its entries go.
struct RowPlace {
  int seen;
  int first;
};

// Of the rows r0 .. of a list, lane i's.  (All lanes of a wavefront call.)
__device__ __forceinline__ RowPlace place_of_row(const SelectArgs &a, long long list, long long r0, int lane) {
  const long long b = (unsigned)list / (unsigned)a.heads, h = list - b * a.heads, r = r0 + lane;
  if (a.blocks) {
    long long before = 0;
    for (long long i = lane; i < b; i += 64) before += min(max(0ll, min((long long)a.blocks[i], a.columns)), a.count);
    for (int o = 1; o < 64; o <<= 1) before += __shfl_xor(before, o, 64);
    const long long seen = max(0ll, min((long long)a.blocks[b], a.columns));
    return {(int)seen, (int)(before * a.heads * a.rows + (h * a.rows + r) * min(seen, a.count))};
  }
  const long long seen = r < a.rows ? blocks_seen(a, r) : 0;
  int mine = (int)min(seen, a.count), upto = mine;
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o, 64);
    if (lane >= o) upto += x;
  }
  return {(int)seen, (int)(list * a.list_entries + entries_before(a, r0)) + upto - mine};
}

// The page or block that column j of list (b, h) stands for; -1: none.
__device__ __forceinline__ long long row_of_codes(const SelectArgs &a, long long b, long long j) {
  if (!a.table) return j;
  const long long page = a.table[b * a.table_width + j];
  return page >= 0 && page < a.pages ? page : -1;
}

__device__ __forceinline__ unsigned wave_max(unsigned v) {
  v = group_max<16>(v);
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  const unsigned a = max((unsigned)p[0], (unsigned)p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return max((unsigned)q[0], (unsigned)q[1]);
}

// Set bits of a mask below this lane's.
__device__ __forceinline__ int lanes_below(unsigned long long mask) {
  return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}

constexpr unsigned kTaken = 0xffffffffu;  // key of a block that is taken whatever it scores

// The `need` best of `seen` keys, fewer than seen; `key(i)` is this lane's key of block 64 i + lane (0 from `seen` on), NV > 0: i
// below NV, from registers.  A threshold that leaves `need` blocks at or above it is searched for from the best score down,
// half an octave, two, eight ... of scores away, then by halving; the largest that leaves more, if none leaves as many.  (Bit
// by bit over the whole range took twice as many steps: most of them went through exponents that no score has.)
// Equal keys at the threshold are taken from the lowest block on.
template <int NV, typename Key>
__device__ __forceinline__ void take_best(int seen, int need, int *out, int lane, const int *__restrict__ table, Key key) {
  const int steps = NV ? NV : (seen + 63) / 64;
  unsigned most = 0;
#pragma unroll NV ? NV : 1
  for (int i = 0; i < steps; ++i) {
    const unsigned k = key(i);
    most = max(most, k == kTaken ? 0u : k);
  }
  most = __builtin_amdgcn_readfirstlane(wave_max(most));
  const auto at_least = [&](unsigned candidate) {
    int n = 0;
#pragma unroll NV ? NV : 1
    for (int i = 0; i < steps; ++i) n += __popcll(__ballot(key(i) >= candidate));
    return n;
  };
  unsigned threshold = 0, beyond = most + 1;  // too few are at or above `beyond`, or just as many
  int at_or_above = seen;
  const int taken_anyway = at_least(beyond);
  if (taken_anyway >= need) {
    threshold = beyond;
    at_or_above = need;
  } else {
    for (unsigned step = 1u << 22; step != 0 && most > step; step <<= 2) {
      const int n = at_least(most - step);
      if (n >= need) {
        threshold = most - step;
        at_or_above = n;
        break;
      }
      beyond = most - step;
    }
    while (at_or_above != need && beyond - threshold > 1) {
      const unsigned middle = threshold + (beyond - threshold) / 2;
      const int n = at_least(middle);
      if (n >= need) threshold = middle, at_or_above = n;
      else beyond = middle;
    }
  }
  int at = 0;
  const auto put = [&](bool take, int i) {
    const unsigned long long taken = __ballot(take);
    if (take) {
      const int j = i * 64 + lane;
      out[at + lanes_below(taken)] = table ? table[j] : j;
    }
    at += __popcll(taken);
  };
  if (at_or_above == need && threshold > 0) {
#pragma unroll NV ? NV : 1
    for (int i = 0; i < steps; ++i) put(key(i) >= threshold, i);
    return;
  }
  int above = 0;
#pragma unroll NV ? NV : 1
  for (int i = 0; i < steps; ++i) above += __popcll(__ballot(key(i) > threshold));
  int equal_left = need - above;  // of the blocks at the threshold itself
#pragma unroll NV ? NV : 1
  for (int i = 0; i < steps; ++i) {
    const unsigned k = key(i);
    const bool equal = i * 64 + lane < seen && k == threshold;
    const unsigned long long ties = __ballot(equal);
    const bool take = k > threshold || (equal && lanes_below(ties) < equal_left);
    equal_left -= min(__popcll(ties), equal_left);
    put(take, i);
  }
}

__device__ __forceinline__ void take_all(int seen, int *out, int lane, const int *__restrict__ table) {
  for (int j = lane; j < seen; j += 64) out[j] = table ? table[j] : j;
}

// A workgroup takes 16 rows of a list.  Scores come from matrix instructions (16 rows x 16 blocks, 64 codes a step; the
// queries' codes stay in registers), go to LDS as sortable numbers and are taken by a wavefront per row, NV a lane.  The search
// is one chain of compare, count and branch: it takes many wavefronts to fill the time between, and 64 rows a workgroup, which
// read the codes of K a quarter as often, left room for a quarter of them (174 us against 96 for 131 072 rows of up to 256).
// Since then 79 us for those rows, dim 128: bound by vector instructions, about 300 a row, 72 % of the cycles.
template <int NV, int KC>
__global__ __launch_bounds__(256) void block_select_kernel(SelectArgs a, long long tiles_of_list) {
  constexpr int RT = 16, STRIDE = NV * 64 + 4;  // rows four apart start 16 banks apart
  __shared__ unsigned keys[RT][STRIDE];
  __shared__ RowPlace places[RT];
  __shared__ int most_seen;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, quarter = lane >> 4;
  const long long block = xcd_contiguous_block(linear_block(), gridDim.x * gridDim.y);
  // (the grid has fewer than 2^32 workgroups)
  const long long list = (unsigned)block / (unsigned)tiles_of_list, r0 = (block - list * tiles_of_list) * RT;
  const long long b = (unsigned)list / (unsigned)a.heads, h = list - b * a.heads;
  if (list >= a.batch * a.heads) return;
  const int rows = (int)min((long long)RT, a.rows - r0);
  if (wave == 0) {
    const RowPlace p = place_of_row(a, list, r0, lane);
    if (lane < RT) places[lane] = p;
    const unsigned top = group_max<64>(lane < rows ? (unsigned)p.seen : 0u);
    if (lane == 0) most_seen = (int)top;
    const long long row = list * a.rows + r0 + lane;
    if (lane < rows) {
      a.pos[row] = p.first;
      if (row == a.batch * a.heads * a.rows - 1) a.pos[row + 1] = p.first + (int)min((long long)p.seen, a.count);
    }
  }
  v4i qf[RT / 16][KC];
#pragma unroll
  for (int x = 0; x < RT / 16; ++x)
#pragma unroll
    for (int s = 0; s < KC; ++s) {
      const int r = 16 * x + col, d = 64 * s + 16 * quarter;
      qf[x][s] = v4i{0, 0, 0, 0};
      if (r < rows) {
        const signed char *q = a.q + (list * a.rows + r0 + r) * a.dim + d;
        if (d < a.dim) *(v2i *)&qf[x][s] = *(const v2i *)q;
        if (d + 8 < a.dim) ((v2i *)&qf[x][s])[1] = *(const v2i *)(q + 8);
      }
    }
  __syncthreads();
  const int seen_all = most_seen;
  if (seen_all > a.count)  // else every row takes what it sees
    for (int j0 = wave * 16; j0 < seen_all; j0 += 64) {
      const int j = j0 + col;
      const long long from = j < seen_all ? row_of_codes(a, b, j) : -1;
      float scale = __builtin_nanf("");
      v4i kf[KC];
#pragma unroll
      for (int s = 0; s < KC; ++s) kf[s] = v4i{0, 0, 0, 0};
      if (from >= 0) {
        const signed char *k = a.k + h * a.k_stride[1] + from * a.k_stride[2] + (a.table ? 0 : b * a.k_stride[0]);
        scale = a.scales[h * a.scale_stride[1] + from * a.scale_stride[2] + (a.table ? 0 : b * a.scale_stride[0])];
#pragma unroll
        for (int s = 0; s < KC; ++s) {
          const int d = 64 * s + 16 * quarter;
          if (d < a.dim) *(v2i *)&kf[s] = *(const v2i *)(k + d);
          if (d + 8 < a.dim) ((v2i *)&kf[s])[1] = *(const v2i *)(k + d + 8);
        }
      }
#pragma unroll
      for (int x = 0; x < RT / 16; ++x) {
        v4i dot = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KC; ++s) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf[x][s], kf[s], dot, 0, 0, 0);
        if (__any(abs_bits(scale) >= kInfBits)) {  // only then is there a NaN
#pragma unroll
          for (int e = 0; e < 4; ++e) keys[16 * x + 4 * quarter + e][j] = sortable((float)dot[e] * scale);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) keys[16 * x + 4 * quarter + e][j] = sortable_number((float)dot[e] * scale);
        }
      }
    }
  __syncthreads();
  const int *table = a.table ? a.table + b * a.table_width : nullptr;
  for (int r = wave; r < rows; r += 4) {
    const int seen = places[r].seen, need = (int)min((long long)seen, a.count);
    int *out = a.crd + places[r].first;
    if (need == seen) {
      take_all(seen, out, lane, table);
      continue;
    }
    const int sink = (int)a.sink, local = (int)a.local;
    for (int x = lane; x < sink + local; x += 64) keys[r][x < sink ? x : seen - local + x - sink] = kTaken;
    wave_lds_sync();
    unsigned k[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) k[i] = i * 64 + lane < seen ? keys[r][i * 64 + lane] : 0u;
    take_best<NV>(seen, need, out, lane, table, [&](int i) { return k[i]; });
  }
}

// Rows of more blocks or longer codes than that: scores go through memory, one wavefront per row, `rows` of them from row0 on.
__global__ __launch_bounds__(64) void block_select_long_kernel(SelectArgs a, unsigned *scores, long long row0, long long rows) {
  const long long at = linear_block(), row = row0 + at;
  const int lane = threadIdx.x;
  if (at >= rows) return;  // workgroups past the count asked for have no scores of their own
  const long long list = row / a.rows, b = list / a.heads, h = list - b * a.heads;
  RowPlace p = place_of_row(a, list, row - list * a.rows, lane);
  p.seen = __builtin_amdgcn_readfirstlane(p.seen);
  p.first = __builtin_amdgcn_readfirstlane(p.first);
  const int need = (int)min((long long)p.seen, a.count);
  if (lane == 0) {
    a.pos[row] = p.first;
    if (row == a.batch * a.heads * a.rows - 1) a.pos[row + 1] = p.first + need;
  }
  const int *table = a.table ? a.table + b * a.table_width : nullptr;
  if (need == p.seen) {
    take_all(p.seen, a.crd + p.first, lane, table);
    return;
  }
  unsigned *mine = scores + at * a.columns;  // a lane reads what it has written itself
  const signed char *q = a.q + row * a.dim;
  for (long long j = lane; j < p.seen; j += 64) {
    unsigned key = kTaken;
    if (j >= a.sink && j < p.seen - a.local) {
      const long long from = row_of_codes(a, b, j);
      float score = __builtin_nanf("");
      if (from >= 0) {
        const signed char *k = a.k + h * a.k_stride[1] + from * a.k_stride[2] + (a.table ? 0 : b * a.k_stride[0]);
        int dot = 0;
        for (int d = 0; d < a.dim; d += 8) {
          const v2i x = *(const v2i *)(q + d), y = *(const v2i *)(k + d);
          dot = __builtin_amdgcn_sdot4(x[0], y[0], dot, false);
          dot = __builtin_amdgcn_sdot4(x[1], y[1], dot, false);
        }
        score = (float)dot * a.scales[h * a.scale_stride[1] + from * a.scale_stride[2] + (a.table ? 0 : b * a.scale_stride[0])];
      }
      key = sortable(score);
    }
    mine[j] = key;
  }
  take_best<0>(p.seen, need, a.crd + p.first, lane, table, [&](int i) { return i * 64 + lane < p.seen ? mine[i * 64 + lane] : 0u; });
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
  set_stretches(a);
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
  block = std::min(block, std::max(tokens, INT64_C(1)));  // a longer one has no more tokens
  PoolArgs a = {static_cast<char *>(x->data), {x->stride[0], x->stride[1], x->stride[2]}, tokens, ceil_div(tokens, block),
                batch * groups * ceil_div(tokens, block), block, (int)groups, (int)(heads / groups), (int)dim, (signed char *)codes, scales};
  if (a.lists_blocks == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(codes && scales && (x->data || heads == 0), "block_pool: null operands");  // the mean of no heads is not a number
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

namespace lapis {
namespace {

constexpr int kShortColumns = 2048, kShortDim = 256;
constexpr int64_t kScoreBytes = INT64_C(256) << 20;  // of rows that go through memory at a time

bool short_rows(const SelectArgs &a) { return a.columns <= kShortColumns && a.dim <= kShortDim; }

// Rows at a time of those that go through memory.
long long rows_at_once(const SelectArgs &a) { return std::max<int64_t>(1, std::min<int64_t>(a.batch * a.heads * a.rows, kScoreBytes / (4 * std::max(a.columns, 1ll)))); }

template <int NV>
void launch_select(const SelectArgs &a, hipStream_t st) {
  const long long tiles = ceil_div(a.rows, 16);
  const dim3 grid = grid_of(a.batch * a.heads * tiles);
  if (a.dim <= 64) hipLaunchKernelGGL((block_select_kernel<NV, 1>), grid, dim3(256), 0, st, a, tiles);
  else if (a.dim <= 128) hipLaunchKernelGGL((block_select_kernel<NV, 2>), grid, dim3(256), 0, st, a, tiles);
  else hipLaunchKernelGGL((block_select_kernel<NV, 4>), grid, dim3(256), 0, st, a, tiles);
}

}  // namespace
}  // namespace lapis

extern "C" int lapis_hip_block_select_work(const lapis_hip_select_args *args, int64_t *bytes) {
  SelectArgs a;
  const int rc = read_select("block_select", args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "block_select: null result");
  *bytes = short_rows(a) ? 0 : 4 * a.columns * rows_at_once(a);
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
    LAPIS_REQUIRE(a.q && a.k && a.scales && a.crd, "block_select: null operands");
    LAPIS_REQUIRE(short_rows(a) || (args->work && aligned16(args->work)), "block_select: work that is null or not on a 16-byte boundary");
    const uintptr_t low = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k);
    LAPIS_REQUIRE((low & 7u) == 0 && strides_of_8(args->k_stride, 3), "block_select: codes that are not on 8-byte boundaries or strides that are no multiples of 8");
  }
  const hipStream_t st = as_stream(stream);
  if (!short_rows(a)) {
    const long long some = rows_at_once(a);
    for (long long row0 = 0; row0 < rows; row0 += some) {
      const long long here = std::min(some, rows - row0);
      hipLaunchKernelGGL(block_select_long_kernel, grid_of(here), dim3(64), 0, st, a, static_cast<unsigned *>(args->work), row0, here);
    }
  } else if (a.columns <= 256) {
    launch_select<4>(a, st);
  } else if (a.columns <= 512) {
    launch_select<8>(a, st);
  } else if (a.columns <= 1024) {
    launch_select<16>(a, st);
  } else {
    launch_select<32>(a, st);
  }
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}
