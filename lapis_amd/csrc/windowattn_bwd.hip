// Attention over a window and the first keys, backward: dK and dV, and the calls.
//
// P and dS are computed twice, once beside dQ (along the queries, with the kernels of attention over lists) and once here, along the
// keys: nothing is added by atomics, so the same inputs give the same bits.
#include "blockattn.hpp"

namespace lapis {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 128;  // of a column

// Columns of 128 keys and their work.  A list has `sink_columns` columns of first keys, whose queries are those that the keys' windows have left
// behind, and after them the columns of all keys, with the queries whose windows hold them.  The work of a column is its queries and
// `overhead` (what a column costs by itself, in queries).  Workgroup i takes i * chunk up to (i + 1) * chunk of all lists' columns one
// behind the other, so that all have the same to do; what a column gets from several places is joined afterwards, in their order.
struct WindowColumns {
  int lists, columns, sink_columns, overhead;
  int queries, shift, window;
  long long of_list, all, chunk;
  int workgroups;
  bool whole;  // a cut in a column of all keys moves to its nearer end: such columns are one workgroup's each
  // Of each workgroup dk and dv of the column that it begins in the middle of, and of the one that it leaves unfinished; behind them, of each
  // list, those of whole columns that first keys are in: sink_columns of first keys, as many of all keys.
  float *partial;

  // Sum over i < c of 128 i + a, cut to 0 .. queries.
  __host__ __device__ long long sum(int c, long long a) const {
    const auto reaches = [&](long long x) {  // first i with 128 i + a >= x
      const long long i = (x - a + kKeys - 1) >> 7;
      return i < 0 ? 0 : i > c ? c : (int)i;
    };
    const int lo = reaches(0), hi = reaches(queries);
    return 64 * ((long long)hi * (hi - 1) - (long long)lo * (lo - 1)) + a * (hi - lo) + (long long)(c - hi) * queries;
  }
  // Work of a list's first k columns.
  __host__ __device__ long long before(int k) const {
    const int sinks = k < sink_columns ? k : sink_columns, c = k - sinks;
    return (long long)sinks * queries - sum(sinks, (long long)window - shift) + sum(c, (long long)window + kKeys - 1 - shift) - sum(c, -(long long)shift) +
           (long long)k * overhead;
  }
  // The queries of a column of a list: from `first` on, these many.
  __device__ __forceinline__ void queries_of(int k, int *first, int *count) const {
    const bool sinks = k < sink_columns;
    const long long low = (long long)(sinks ? k : k - sink_columns) * kKeys - shift + (sinks ? window : 0);
    const long long end = sinks ? queries : low + kKeys - 1 + window;
    const long long from = low < 0 ? 0 : low > queries ? queries : low, to = end < 0 ? 0 : end > queries ? queries : end;
    *first = (int)from;
    *count = (int)(to - from);
  }
};

__device__ __forceinline__ long long same_lane(long long x, int lane) {
  return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, lane));
}
// Column k of list `list`, from `start` up to `end` of all work.
struct Column {
  int list, k;
  long long start, end;
};
// The column that a place in all work belongs to: a wavefront looks at 64 candidates a step.
__device__ __forceinline__ Column find_column(const WindowColumns &t, long long at, int lane) {
  Column c;
  c.list = (int)((double)at / (double)t.of_list);
  if (c.list * t.of_list > at) --c.list;
  if ((c.list + 1) * t.of_list <= at) ++c.list;
  const long long in = at - c.list * t.of_list;
  int lo = 0, n = t.sink_columns + t.columns;
  for (;;) {
    const int step = (n + 62) / 63, k = min(lo + lane * step, lo + n);  // up to the first one behind them
    const long long from = t.before(k);
    const int pick = 63 - __clzll(__ballot(from <= in && k < lo + n));
    if (step == 1) {
      c.k = lo + pick;
      c.start = c.list * t.of_list + same_lane(from, pick);
      c.end = c.list * t.of_list + same_lane(from, pick + 1);
      return c;
    }
    lo += pick * step;
    n = min(step, n - pick * step);
  }
}

// Where the work of workgroup w begins, and that of the one before ends.
__device__ __forceinline__ long long cut_of(const WindowColumns &t, long long w, int lane) {
  const long long at = w * t.chunk;
  if (!t.whole || at >= t.all) return min(at, t.all);
  const Column c = find_column(t, at, lane);
  return c.k < t.sink_columns ? at : at - c.start < c.end - at ? c.start : c.end;
}

// Row `row` (the same for all lanes) of a 32x32 product that has been rounded to an operand, in its column's lanes of both halves.
template <typename T>
__device__ __forceinline__ float of_row(const vec8<T> (&f)[2], int row, int lane) {
  float w = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) w = (row & ~4) == 8 * (e >> 2) + (e & 3) ? (float)f[e >> 3][e & 7] : w;
  return __shfl(w, (lane & 31) | (row & 4) << 3, 64);
}

template <typename T, int DP>
struct DkvLds {
  static constexpr int ROWS = 64;  // of a stage: a tile of 32 for each half of the wavefronts
  __attribute__((aligned(256))) typename T::elem kv[2][kKeys * DP];       // keys and values, rows in the order of place_of
  __attribute__((aligned(256))) typename T::elem tiles[2][2][ROWS * DP];  // two stages of queries and dO
  __attribute__((aligned(16))) float sums[2][2][ROWS];                    // log-sums and deltas of a stage's rows
  __attribute__((aligned(16))) int position[2][ROWS];                     // of its rows; -1: no row
  int bad;
};

struct DkvArgs {
  BlockArgs a;
  WindowColumns cols;
  const float *delta, *logs;
};
// The arguments are more than the scalar registers hold beside the loop: what it does not need is read again where it is used.
typedef const __attribute__((address_space(4))) DkvArgs *DkvArgsAgain;
__device__ __forceinline__ const DkvArgs &again() {
  DkvArgsAgain p = (DkvArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const DkvArgs *)p;
}

// 8192 queries and keys, 32 heads over 8, dim 128, window 1024 and the first 16 keys, bf16: 406 us in a trace (364 at best), 645 to 700 TFLOP/s of its four
// products, and 20 for the join.  Bound by the card's power: products run in 40 % of the cycles, LDS in 37 %, other orders of the work take the same time
// (weights of half a tile under the products of the other half too), and the whole pass a quarter less with operands that are zeros.  3 x 701 queries, 937 keys, 6 heads, dim 72, window 200: 31 us, of
// which a first stage takes 8 (launch, instructions and operands from memory) and each stage of 64 rows 2.5.
//
// 128 keys of a list and a stretch of the queries that see them, rows (a query times a head of the group) packed into tiles of 32.
// Four wavefronts have 32 keys each, a key per lane, and four more the same keys and every other tile: a wavefront computes all four
// products of its tile, S = Q K^T and dP = dO V^T, which turn into P and dS and feed dV^T = dO^T P and dK^T = Q^T dS from their
// registers, each rounded once to the operands' type (products of 32-bit operands have a sixteenth of the rate), and the halves' sums are added up at the
// column's end.
// Two wavefronts a SIMD, one in its products while the other is in its weights: with one alone (K and V in its registers, three tiles
// in work at a time) each of its 440 instructions a tile took its turn, 3400 cycles where the products take 1100; the sums leave no
// registers for K and V of 32 keys in two, so they are read from LDS, beside the queries.
template <typename T, int DP>
__global__ __launch_bounds__(512, 2) void window_dkv_kernel(DkvArgs) {
  typedef typename T::elem elem;
  typedef DkvLds<T, DP> Lds;
  typedef const __attribute__((address_space(3))) vec8<T> *Rows;
  typedef short s4 __attribute__((ext_vector_type(4)));
  constexpr int PIECES = DP / 8, RP = 512 / PIECES, PASSES = Lds::ROWS / RP, DT = DP / 32, N = DP / 16;
  constexpr unsigned ROW = 2 * DP, ONE = Lds::ROWS * ROW, STAGE = 2 * ONE, VALUES = kKeys * ROW;  // bytes: a row, a stage's queries, a stage, from K to V
  __shared__ Lds mem;
  static_assert(offsetof(Lds, kv) == 0 && offsetof(Lds, tiles) == 2 * VALUES && sizeof(mem.tiles) == 2 * STAGE, "keys, values and stages are cleared together");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int kg = wave & 3, rg = wave >> 2;  // which keys, which tiles
  const int w = (int)xcd_contiguous_block(blockIdx.x, gridDim.x), group = again().a.group, dim = again().a.dim;
  const float scale = again().a.scale, c = scale * kLog2e;

  // Where this lane's operands lie: piece p of its row, and of its four rows of columns, is an exclusive or away from the first.  (Made anew in each
  // tile, or the compiler keeps all of them in registers.)
  const unsigned kv_at = lds_address(mem.kv[0]), tiles_at = lds_address(mem.tiles[0][0]);
  const unsigned row_in = 2 * place_of<DP>(lane & 31, half);
  const int column_row = 4 * half + ((lane & 15) >> 2), column_d = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  unsigned key_row = kv_at + kg * 32 * ROW + row_in, query_row = tiles_at + rg * 32 * ROW + row_in;
  unsigned column_at = tiles_at + rg * 32 * ROW + 2 * (place_of<DP>(column_row, column_d >> 3) + (column_d & 7));
  const auto rows_of = [&](unsigned at, int y, unsigned more) { return *(Rows)(uintptr_t)((at ^ (32u * y)) + more); };
  const auto columns_of = [&](int y, unsigned more) {  // 32 columns from 32 (y % DT) on, of rows 16 (y / DT) ..
    const unsigned at = column_at ^ (64u * (y % DT)), rows = 16 * (y / DT) * ROW;
    const auto read = [&](unsigned x) {
      return __builtin_bit_cast(vec4<T>, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(uintptr_t)x));
    };
    return join<T>(read(at + rows + more), read((at ^ 32u) + rows + 8 * ROW + more));  // (row + 8: the other bit of its turn)
  };

  const long long work_start = cut_of(again().cols, w, lane), work_end = cut_of(again().cols, w + 1ll, lane);
  for (long long work = work_start; work < work_end;) {
    const DkvArgs &args = again();
    const BlockArgs &a = args.a;
    const WindowColumns &cols = args.cols;
    const Column of = find_column(cols, work, lane);
    const int bh = of.list, k = of.k, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
    const bool sinks = k < cols.sink_columns;
    const int column = sinks ? k : k - cols.sink_columns;
    const bool begins = work == of.start, ends = of.end <= work_end;
    int first, queries;
    cols.queries_of(k, &first, &queries);
    const int skipped = (int)min((long long)queries, max(0ll, work - of.start - cols.overhead));  // queries of the column that others have
    work = min(of.end, work_end);
    queries = (int)min((long long)queries, max(0ll, work - of.start - cols.overhead)) - skipped;
    first += skipped;
    // Rows, and stages of them.  A row at position p sees a key where p - key is at least `reach` and less than `reach` + `range`.
    const int total = queries * group, stages = total / Lds::ROWS + (total % Lds::ROWS != 0);
    const int reach = sinks ? cols.window : 0;
    const unsigned range = sinks ? 0x40000000u : (unsigned)cols.window;
    const int all_low = column * kKeys, key_low = all_low + kg * 32, key = key_low + (lane & 31), key_reach = key + reach;
    const bool live = key < (sinks ? min(a.sink, a.keys) : a.keys);

    // Rows of stage t start at head 64 t % group of query 64 t / group, which `at_position` and `at_h` count on, a stage at a time.  Where this
    // thread's pieces of a stage lie from that query on, and (wavefronts 0 to 2) its row's sums and position; the same for all stages where
    // group divides 64.
    const int step_q = Lds::ROWS / group, step_h = Lds::ROWS % group, place = tid % PIECES, my_row = tid / PIECES;
    const elem *q_from = (const elem *)a.q.data + b * a.q.stride[0] + first * a.q.stride[1] + kh * group * a.q.stride[2];
    const elem *g_from = (const elem *)a.dout.data + b * a.dout.stride[0] + first * a.dout.stride[1] + kh * group * a.dout.stride[2];
    const float *sums_from = (wave == 0 ? args.logs : args.delta) + (b * a.heads + kh * group) * a.queries + first;
    const long long q_stride = a.q.stride[1], g_stride = a.dout.stride[1];
    unsigned q_off[PASSES], g_off[PASSES], sum_off, own_q;
    int at_h = 0, at_position = first + a.shift, rows = total;
    const auto place_rows = [&]() {  // a row that is not there is read from the stage's first one, and has no weight
      const BlockArgs &a = again().a;
      const unsigned q_heads = (unsigned)a.q.stride[2] * 2, g_heads = (unsigned)a.dout.stride[2] * 2;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const unsigned row = p * RP + my_row, r = at_h + ((int)row < rows ? row : 0), q = r / (unsigned)group, h = r - q * group;
        const unsigned d = (place ^ turn<DP>(row)) * 16;
        q_off[p] = q * ((unsigned)q_stride * 2) + h * q_heads + d;
        g_off[p] = q * ((unsigned)g_stride * 2) + h * g_heads + d;
      }
      const unsigned r = at_h + (lane < rows ? lane : 0);
      own_q = r / (unsigned)group;
      sum_off = ((r - own_q * group) * a.queries + own_q) * 4;
    };
    const auto load = [&](int slot) {  // the stages one after the other
      if (step_h || rows < Lds::ROWS) place_rows();
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const unsigned to = __builtin_amdgcn_readfirstlane(tiles_at + slot * STAGE + (p * 8 + wave) * 1024);
        if ((place ^ turn<DP>(p * RP + my_row)) * 8 < dim) {
          load_to_lds(q_from, q_off[p], to);
          load_to_lds(g_from, g_off[p], to + ONE);
        }
      }
      if (wave < 2) load_word_to_lds(sums_from, sum_off, __builtin_amdgcn_readfirstlane(lds_address(mem.sums[slot][wave])));
      else if (wave == 2) mem.position[slot][lane] = lane < rows ? at_position + (int)own_q : -1;
      int more = step_q;
      if (step_h) {
        at_h += step_h;
        if (at_h >= group) at_h -= group, ++more;
      }
      at_position += more;
      rows -= Lds::ROWS;
      q_from += more * q_stride;
      g_from += more * g_stride;
      sums_from += more;
    };

    __syncthreads();  // the column before
    if (dim < DP)     // what no row fills stays zero
      for (int i = tid; i < (int)(2 * STAGE + 2 * VALUES) / 16; i += 512) ((v4i *)&mem)[i] = v4i{0, 0, 0, 0};
    if (tid == 0) mem.bad = -1;
    __syncthreads();
    if (stages > 0) {
      place_rows();
      load(0);
#pragma unroll
      for (int p = 0; p < kKeys / RP; ++p) {
        const int row = p * RP + my_row, d = (place ^ turn<DP>(row)) * 8;
        const long long from = min(all_low + row, a.keys - 1);  // (keys that are not there are not asked for)
        const unsigned to = __builtin_amdgcn_readfirstlane(kv_at + (p * 8 + wave) * 1024);
        if (d < dim) {
          load_to_lds((const elem *)a.k.data + b * a.k.stride[0] + from * a.k.stride[1] + kh * a.k.stride[2] + d, to);
          load_to_lds((const elem *)a.v.data + b * a.v.stride[0] + from * a.v.stride[1] + kh * a.v.stride[2] + d, to + VALUES);
        }
      }
    }
    lds_loads_done();

    // Some row of 32 (a tile) does not see some key of low .. low + n - 1 (of first keys: those that are) where the tile's first position is too
    // near to the last of them, where its last one is too far from the first, and where rows are missing: up to some tile, and from another on.
    const auto uncut = [&](int low, int n, int *begin, int *end) {
      const long long base = first + a.shift, last_key = (sinks ? min(low + n, a.sink) : low + n) - 1;
      *begin = (int)max(0ll, min(((last_key + reach - base) * group + 31) >> 5, (1ll << 30)));
      *end = (int)max(0ll, min(((long long)low + reach + range - base) * group >> 5, (long long)total >> 5));
    };
    int from_tile, to_tile, all_from, all_to;
    uncut(key_low, 32, &from_tile, &to_tile);
    uncut(all_low, kKeys, &all_from, &all_to);
    const auto sees_key = [&](int position) { return (unsigned)(position - key_reach) < range; };

    v16f accv[DT], acck[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) accv[i] = acck[i] = v16f{};
    // Rows that some mask of the workgroup cuts and that hold an infinity or NaN: those elements count for the keys that their rows see, by
    // themselves, and the products take them as zeros.
    const auto mend = [&](int slot, const vec8<T> (&p)[2], const vec8<T> (&ds)[2]) {
      const int *at = mem.position[slot] + 32 * rg;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const elem *tile = mem.tiles[slot][which] + 32 * rg * DP;
        unsigned bad_rows = 0;
#pragma unroll 1
        for (int i = 0; i < PIECES / 2; ++i) {
          const unsigned long long lanes = __ballot(not_finite<T>(*(const vec8<T> *)(tile + (i * 64 + lane) * 8)));
#pragma unroll
          for (int x = 0; x < 64 / PIECES; ++x)
            if (lanes >> (x * PIECES) & ((1u << PIECES) - 1)) bad_rows |= 1u << (i * (64 / PIECES) + x);
        }
        bad_rows = __builtin_amdgcn_readfirstlane(bad_rows);
#pragma unroll 1
        for (; bad_rows != 0; bad_rows &= bad_rows - 1) {
          const int row = __builtin_ctz(bad_rows);
          const float by = which ? of_row<T>(p, row, lane) : of_row<T>(ds, row, lane);
          const bool sees = sees_key(at[row]);
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const vec4<T> x = *(const vec4<T> *)(tile + place_of<DP>(row, 4 * i + (e >> 2)) + 4 * half);
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                const float y = (float)x[n];
                if (sees && abs_bits(y) >= kInfBits) {
                  if (which) accv[i][e + n] += by * y;
                  else acck[i][e + n] += by * y;
                }
              }
            }
        }
      }
      __syncthreads();
      for (int i = tid; i < (int)STAGE / 16; i += 512) {
        vec8<T> *x = (vec8<T> *)mem.tiles[slot][0] + i;
        *x = finite_only<T>(*x);
      }
      __syncthreads();
    };
    __syncthreads();

    const auto step = [&](int t, auto which) {
      constexpr int slot = decltype(which)::value;
      constexpr unsigned at = slot * STAGE;
      const int tile = 2 * t + rg;
      asm volatile("" : "+v"(key_row), "+v"(query_row), "+v"(column_at));
      if (t + 1 < stages) load(1 - slot);
      const bool looks = 2 * t < all_from || 2 * t + 2 > all_to;
      if (looks) {
        bool bad = false;
        for (int i = tid; i < (int)STAGE / 16; i += 512) bad |= not_finite<T>(*((const vec8<T> *)mem.tiles[slot][0] + i));
        if (__any(bad) && lane == 0) mem.bad = t;
        __syncthreads();
      }
      // scores, their operands read some products ahead
      constexpr int AHEAD = 2;
      v16f s = {}, g = {};
      {
        vec8<T> qa[N], ka[N], ga[N], va[N];
        const auto read = [&](int y) {
          qa[y] = rows_of(query_row, y, at);
          ka[y] = rows_of(key_row, y, 0);
          ga[y] = rows_of(query_row, y, at + ONE);
          va[y] = rows_of(key_row, y, VALUES);
        };
#pragma unroll
        for (int y = 0; y < AHEAD; ++y) read(y);
        const auto score = [&](int y) {
          if (y + AHEAD < N) read(y + AHEAD);
          s = mfma32(qa[y], ka[y], s);
          g = mfma32(ga[y], va[y], g);
          __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int y = 0; y < N * 3 / 4; ++y) score(y);
        if (DP <= 64 || dim > 96) {  // the last quarter of a row, if it is there (dim 96, 8192 queries, window 1024: 635 us with dQ's, 595 without)
#pragma unroll
          for (int y = N * 3 / 4; y < N; ++y) score(y);
        }
      }
      vec8<T> p[2], ds[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4f off = *(const v4f *)(mem.sums[slot][0] + 32 * rg + 8 * j + 4 * half), del = *(const v4f *)(mem.sums[slot][1] + 32 * rg + 8 * j + 4 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 4 * j + i;
          const float by = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -off[i]));
          p[e >> 3][e & 7] = (elem)by;
          ds[e >> 3][e & 7] = (elem)(by * __builtin_fmaf(g[e], scale, -del[i]));
        }
      }
      if (tile < from_tile || tile >= to_tile) {  // no weight for what a row does not see, whatever its numbers are
        asm volatile("");                         // (a branch, not selects)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const v4i pos = *(const v4i *)(mem.position[slot] + 32 * rg + 8 * j + 4 * half);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned keep = (sees_key(pos[2 * i]) ? 0xffffu : 0u) | (sees_key(pos[2 * i + 1]) ? 0xffff0000u : 0u);
            const auto cut = [&](vec8<T> &x) {
              v4u words = __builtin_bit_cast(v4u, x);
              words[2 * (j & 1) + i] &= keep;
              x = __builtin_bit_cast(vec8<T>, words);
            };
            cut(p[j >> 1]);
            cut(ds[j >> 1]);
          }
        }
      }
      if (looks && mem.bad == t) mend(slot, p, ds);
      {
        constexpr int LAST = DP <= 64 ? 0 : N / DT, FIRST = N - LAST;  // products of the last 32 columns come last
        const auto row_of = [](int y) { return y < FIRST ? y / (FIRST * DT / N) : y - FIRST; };
        const auto column_of = [](int y) { return y < FIRST ? y % (FIRST * DT / N) : DT - 1; };
        vec8<T> xg[N], xq[N];
        const auto read = [&](int y) {
          xg[y] = columns_of(row_of(y) * DT + column_of(y), at + ONE);
          xq[y] = columns_of(row_of(y) * DT + column_of(y), at);
        };
        const auto products = [&](int y) {
          if (y + AHEAD < N) read(y + AHEAD);
          accv[column_of(y)] = mfma32(xg[y], p[row_of(y)], accv[column_of(y)]);
          acck[column_of(y)] = mfma32(xq[y], ds[row_of(y)], acck[column_of(y)]);
          __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int y = 0; y < AHEAD; ++y) read(y);
#pragma unroll
        for (int y = 0; y < FIRST; ++y) products(y);
        if (LAST && dim > 96) {
#pragma unroll
          for (int y = FIRST; y < N; ++y) products(y);
        }
      }
      lds_loads_done();
      __syncthreads();
    };
    for (int t = 0; t < stages; t += 2) {
      step(t, std::integral_constant<int, 0>());
      if (t + 1 < stages) step(t + 1, std::integral_constant<int, 1>());
    }

    // The halves' sums: dK is added up by the first, dV by the second, with LDS between them.
    float *between = (float *)mem.kv + kg * DT * 1024;
    const auto give = [&](const v16f (&acc)[DT], float *to) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) *(v4f *)(to + (i * 4 + e / 4) * 256 + lane * 4) = v4f{acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]};
    };
    if (rg) give(acck, between);
    else give(accv, between + 4 * DT * 1024);
    __syncthreads();
    if (!live) continue;
    const float *got = between + (rg ? 4 * DT * 1024 : 0);
    const DkvArgs &at_end = again();
    const View &v = rg ? at_end.a.dv : at_end.a.dk;
    const bool partial = !begins || !ends || column < at_end.cols.sink_columns;
    const long long slot = begins && ends ? 2ll * at_end.cols.workgroups + 2 * bh * at_end.cols.sink_columns + k : 2ll * w + begins;
    float *to = at_end.cols.partial + (2 * slot + rg) * (kKeys * DP) + (kg * 32 + (lane & 31)) * DP;
    elem *out = (elem *)v.data + b * v.stride[0] + key * v.stride[1] + kh * v.stride[2];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * i + 2 * e + 4 * half;
        const v4f more = *(const v4f *)(got + (i * 4 + e / 4) * 256 + lane * 4);
        v4f sum;
        vec4<T> x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[j] = (rg ? accv[i][e + j] : acck[i][e + j]) + more[j];
          x[j] = (elem)sum[j];
        }
        if (partial) *(v4f *)(to + d) = sum;
        else if (d < dim) *(vec4<T> *)(out + d) = x;
      }
  }
}

// Columns that several places have a part of: their sums, first keys first, then in the order of the workgroups.  One workgroup for each
// column that first keys are in, and for each place where one workgroup's work ends and the next one's begins: for the column that is cut there,
// if it is the first such place in it.
template <typename T, int DP>
__global__ __launch_bounds__(256) void window_join_kernel(BlockArgs a, WindowColumns cols) {
  typedef typename T::elem elem;
  __shared__ int found_list, found_column;
  __shared__ long long found_from[2], found_to[2];  // workgroups, or a slot of its own
  __shared__ bool found_whole[2];
  const int of_sinks = cols.lists * cols.sink_columns, block = blockIdx.x, lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int list, column = -1;
    if (block < of_sinks) {
      list = block / cols.sink_columns;
      column = block - list * cols.sink_columns;
    } else {
      const long long at = (block - of_sinks + 1) * cols.chunk;
      const Column c = find_column(cols, at, lane);
      list = c.list;
      if (c.k >= 2 * cols.sink_columns && c.start < at && at - cols.chunk <= c.start) column = c.k - cols.sink_columns;
    }
    if (column >= 0) {
      for (int i = column < cols.sink_columns ? 0 : 1; i < 2; ++i) {
        const int k = i ? cols.sink_columns + column : column;
        const long long edge = list * cols.of_list + cols.before(k + (lane & 1)), start = same_lane(edge, 0), end = same_lane(edge, 1);
        const long long w = start / cols.chunk, last = (end - 1) / cols.chunk;
        const bool whole = w == last || (i && cols.whole);
        if (lane == 0) {
          found_whole[i] = whole;
          found_from[i] = whole ? 2ll * cols.workgroups + 2 * list * cols.sink_columns + k : w;
          found_to[i] = whole ? found_from[i] + 1 : last + 1;
        }
      }
    }
    if (lane == 0) found_list = list, found_column = column;
  }
  __syncthreads();
  const int bh = found_list, column = found_column;
  if (column < 0) return;
  const int b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  constexpr int EACH = kKeys * DP;
  for (int x = (blockIdx.y * 256 + threadIdx.x) * 4; x < 2 * EACH; x += gridDim.y * 1024) {
    const bool is_v = x >= EACH;
    const int at = is_v ? x - EACH : x, d = at % DP, key = column * kKeys + at / DP;
    if (key >= a.keys || d >= a.dim) continue;
    v4f sum = {0.f, 0.f, 0.f, 0.f};
    for (int i = column < cols.sink_columns && key < a.sink ? 0 : 1; i < 2; ++i) {
      for (long long w = found_from[i]; w < found_to[i]; w += 4) {  // four on their way, added in order
        v4f y[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const long long of = min(w + n, found_to[i] - 1), slot = found_whole[i] ? of : 2 * of + (of == found_from[i]);
          y[n] = *(const v4f *)(cols.partial + slot * 2 * EACH + x);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[e] += w + n < found_to[i] ? y[n][e] : 0.f;
      }
    }
    const View &v = is_v ? a.dv : a.dk;
    vec4<T> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (elem)sum[e];
    *(vec4<T> *)((elem *)v.data + b * v.stride[0] + key * v.stride[1] + kh * v.stride[2] + d) = o;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------

struct WindowLayout {
  int64_t delta, logs, partial, bytes;
  bool few;  // rows: dQ by 16 of them
  WindowColumns columns;
};

constexpr int kColumnTiles = 6;  // what a column costs beside its tiles (a stage of two takes 2.5 us, a column's loads, start and end 7)
// Of a workgroup.  With 6, 12 and 24: 3 x 701 queries over 937 keys, 6 heads, dim 72, window 200 62, 53 and 67 us; 1024 queries, 16 heads, dim 64, window 100 46, 42
// and 52; 512 queries, 8 heads over 2, dim 128, window 256 42, 47 and 59; 128 queries over 4096 keys, 8 heads, dim 128 82, 100 and 110.
constexpr int kLeastTiles = 12;

int layout_of(BlockArgs *a, WindowLayout *layout) {
  const char *what = "window_attention_backward";
  WindowLayout &l = *layout = {};
  const int cus = std::max(device_cu_count(), 1);
  cut_queries(a, 128);
  const int64_t lists = (int64_t)a->batch * a->kv_heads;
  l.few = lists * a->rows * ceil_div((int64_t)a->block_m * a->group, 128) < cus / 2;  // the forward pass's rule
  if (l.few) cut_queries(a, 16);
  const int64_t row_tiles = ceil_div((int64_t)a->block_m * a->group, l.few ? 16 : 128);
  LAPIS_REQUIRE(lists * a->rows * row_tiles * 256 < (INT64_C(1) << 32), "%s: %lld rows", what, (long long)(lists * a->rows));
  WindowColumns &c = l.columns;
  c.lists = (int)lists;
  c.columns = (int)ceil_div(a->keys, kKeys);
  LAPIS_REQUIRE(lists * c.columns * 256 < (INT64_C(1) << 32), "%s: %lld lists of %lld keys", what, (long long)lists, (long long)a->keys);
  LAPIS_REQUIRE((int64_t)a->queries * a->group < (1 << 29), "%s: %d queries of %d heads", what, a->queries, a->group);
  const int group = std::max(a->group, 1);
  for (const View *v : {&a->q, &a->dout}) {  // the rows of a stage lie within 32-bit offsets: 64 of them from any head of a group on
    for (int i = 1; i < 3; ++i)
      LAPIS_REQUIRE(v->stride[i] >= 0 && v->stride[i] < (1 << 25), "%s: queries or their gradients with a stride of %lld elements", what, v->stride[i]);
    const int64_t last = group + 62, query = last / group;
    const int64_t farthest = std::max(query * v->stride[1] + (last - query * group) * v->stride[2], (query - 1) * v->stride[1] + (group - 1) * v->stride[2]);
    LAPIS_REQUIRE(2 * (farthest + kMaxBlockDim) < (INT64_C(1) << 32), "%s: %d heads of a group with a stride of %lld elements", what, group, v->stride[2]);
  }
  c.queries = a->queries, c.shift = a->shift, c.window = a->window;
  // first keys that some query's window has left behind
  c.sink_columns = (int)ceil_div(std::min(std::max((int64_t)a->keys - a->window, INT64_C(0)), std::min<int64_t>(a->sink, a->keys)), kKeys);
  c.overhead = std::max(1, kColumnTiles * 32 / group);
  c.of_list = c.before(c.sink_columns + c.columns);
  c.all = lists * c.of_list;
  c.chunk = std::max<int64_t>({1, ceil_div(c.all, cus), ceil_div(kLeastTiles * 32, group)});
  c.workgroups = (int)ceil_div(c.all, c.chunk);
  // Few columns, none of them much longer than a workgroup's share: whole columns take a little longer than equal shares would, but need no join (3 x 701
  // queries, 6 heads, window 200: dK and dV 31.3 us and 6.5 for the first keys' join, equal shares 35.8 and 11.4).
  c.whole = lists * c.columns <= cus && 2ll * (a->window + kKeys + c.overhead) <= 3 * c.chunk;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.delta = take(4ll * a->batch * a->heads * a->queries);
  l.logs = take(4ll * a->batch * a->heads * a->queries);
  if (c.all) l.partial = take((2ll * c.workgroups + 2 * lists * c.sink_columns) * 2 * kKeys * (a->dim <= 64 ? 64 : 128) * 4);
  l.bytes = at;
  return LAPIS_HIP_OK;
}

template <typename T, int DP>
int launch_backward(BlockArgs a, char *work, hipStream_t st) {
  WindowLayout l;
  const int rc = layout_of(&a, &l);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(l.bytes == 0 || (work && aligned16(work)), "window_attention_backward: work that is null or not on a 16-byte boundary");
  WindowColumns &c = l.columns;
  float *delta = reinterpret_cast<float *>(work + l.delta), *logs = reinterpret_cast<float *>(work + l.logs);
  c.partial = reinterpret_cast<float *>(work + l.partial);
  if (a.rows && c.lists) launch_window_dq(a, std::is_same<T, Bf16>::value, l.few, delta, logs, st);
  if (c.all) {
    hipLaunchKernelGGL((window_dkv_kernel<T, DP>), dim3((unsigned)c.workgroups), dim3(512), 0, st, DkvArgs{a, c, delta, logs});
    const int joined = c.lists * c.sink_columns + (c.whole ? 0 : c.workgroups - 1);
    if (joined) hipLaunchKernelGGL((window_join_kernel<T, DP>), dim3((unsigned)joined, 16), dim3(256), 0, st, a, c);
  }
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_window_attention_backward_work(const lapis_hip_window_args *args, int64_t *bytes) {
  LAPIS_CHECK_INIT();  // the size goes by the number of compute units
  BlockArgs a;
  int rc = read_window("window_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "window_attention_backward: null result");
  WindowLayout l;
  rc = layout_of(&a, &l);
  *bytes = l.bytes;
  return rc;
}

extern "C" int lapis_hip_window_attention_backward(const lapis_hip_window_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_window("window_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0 || (a.heads == 0 && a.kv_heads == 0)) return LAPIS_HIP_OK;
  char *work = static_cast<char *>(args->work);
  const hipStream_t st = as_stream(stream);
  const bool bf16 = args->dtype == LAPIS_HIP_BF16;
  if (a.dim <= 64) return bf16 ? launch_backward<Bf16, 64>(a, work, st) : launch_backward<F16, 64>(a, work, st);
  return bf16 ? launch_backward<Bf16, 128>(a, work, st) : launch_backward<F16, 128>(a, work, st);
}
