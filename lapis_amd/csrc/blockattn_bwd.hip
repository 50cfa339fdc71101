// Attention over the blocks that a CSR structure lists, or over a window and the first keys, backward.
//
// P and dS are computed twice, once beside dQ (rows of the structure, as in the forward pass) and once beside dK and dV
// (its columns): nothing is added by atomics, so the same inputs give the same bits.  The columns' lists of rows are made
// here (counted, summed, filled: three small kernels), since a selection is another one in every training step.
#include "blockattn.hpp"

namespace lapis {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kParts = 8;  // of the units of work beside dK and dV, one to each XCD

// Row `row` (the same for all lanes) of a 32x32 product that has been rounded to an operand, in its column's lanes of both halves.
template <typename T>
__device__ __forceinline__ float of_row(const vec8<T> (&f)[2], int row, int lane) {
  float w = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) w = (row & ~4) == 8 * (e >> 2) + (e & 3) ? (float)f[e >> 3][e & 7] : w;
  return __shfl(w, (lane & 31) | (row & 4) << 3, 64);  // rows with this bit are in the other half's lanes
}

// ---- dQ --------------------------------------------------------------------------------------------------------

// As the forward kernel: 32 rows a wavefront, a query per lane.  dS^T = P^T * (scale V dO^T - scale delta) feeds dQ^T = K^T dS^T
// from its registers.  rowsum(dO * O), times `scale`, and the log-sums in units of ln 2 are left for the other kernel.
// 8192 queries, 32 heads over 8, dim 128, 16 blocks of 64 a row: 273 us in a trace (309 with a branch for each masked element and operands read where
// they are used, 356 with 24 registers spilled and the products one chain after the other), 690 TFLOP/s; a window of 1024 and the first 16 keys
// 293.  Bound by what a wavefront waits for between its chains of products: they run in a third of the cycles.
// Head dims up to 64: three wavefronts a SIMD, 168 registers, one of them read back from memory once a tile (left to itself the compiler takes 169 and two wavefronts; 1981
// queries, 40 heads over 8, dim 32, 9 blocks of 32: 26.5 us with two, 21.7 with three; 8192 queries, 32 heads, dim 64, 16 blocks of 64: 159 and 143).
template <typename T, int DP, int NW, int KT, bool WINDOW, int SIDES = 1>
__global__ __launch_bounds__(64 * NW * SIDES, DP <= 64 && SIDES == 1 ? 3 : 2) void block_dq_kernel(BlockArgs a, int tiles_of_list, float *__restrict__ delta, float *__restrict__ logs, int *odd) {
  typedef typename T::elem elem;
  constexpr int PIECES = DP / 8, PASSES = KT * PIECES / (NW * 64), ST = KT / 32, DT = DP / 32, CH = KT / 16;
  __shared__ __attribute__((aligned(16))) elem k_tile[SIDES][2][KT * DP], v_tile[SIDES][2][KT * DP];
  __shared__ int bad_tile[SIDES][2];
  const int tid = threadIdx.x % (64 * NW), side = SIDES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * NW)), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const unsigned block = xcd_contiguous_block(blockIdx.x, gridDim.x);
  if (!WINDOW && block == 0 && tid <= kParts) odd[tid] = 0;  // for the kernels after this one: the flag and the counters behind it
  const int list = block / tiles_of_list, part = block - list * tiles_of_list;
  const int bh = list / a.rows, r = list - bh * a.rows, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const int q0 = r * a.block_m, held = min(a.block_m, a.queries - q0), rows = held * a.group;
  if (part * 32 * NW >= rows) return;
  int first = 0, count = 0;
  if (!WINDOW) entries_of(a, list, &first, &count);

  const int row0 = part * 32 * NW + wave * 32, row = row0 + (lane & 31);
  const bool live = row < rows;
  const int query = q0 + row / a.group, head = kh * a.group + row % a.group;
  const int limit = a.causal ? min(query + a.shift, a.keys - 1) : a.keys - 1;
  const int row_last = min(row0 + 31, rows - 1);
  const int low = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row0 / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int high = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row_last / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int low_of_all = a.causal ? min(q0 + part * 32 * NW / a.group + a.shift, a.keys - 1) : a.keys - 1;
  const int row_last_of_all = min(part * 32 * NW + 32 * NW, rows) - 1;
  const Sight<WINDOW> row_sees(a, limit);
  const int gone_any = high - a.window, gone_any_of_all = q0 + row_last_of_all / a.group + a.shift - a.window;

  vec8<T> qf[DP / 16], gf[DP / 16];
  float off = INFINITY, del = 0.f;  // of a row without entries: weights 0
  const elem *qp = (const elem *)a.q.data + b * a.q.stride[0] + query * a.q.stride[1] + head * a.q.stride[2];
  const elem *gp = (const elem *)a.dout.data + b * a.dout.stride[0] + query * a.dout.stride[1] + head * a.dout.stride[2];
  const elem *op = (const elem *)a.out.data + b * a.out.stride[0] + query * a.out.stride[1] + head * a.out.stride[2];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * half;
    vec8<T> o = {};
    qf[s] = gf[s] = vec8<T>{};
    if (live && d < a.dim) {
      qf[s] = *(const vec8<T> *)(qp + d);
      gf[s] = *(const vec8<T> *)(gp + d);
      o = *(const vec8<T> *)(op + d);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) del += (float)gf[s][j] * (float)o[j];
  }
  del = halves_sum(del) * a.scale;
  if (live) {
    const long long at = ((long long)b * a.heads + head) * a.queries + query;
    const float lse = a.lse[at];
    off = lse == -INFINITY ? INFINITY : lse * kLog2e;
    if (half == 0 && side == 0) delta[at] = del, logs[at] = off;
  }
  KeyTiles<T, DP, NW, KT, false, WINDOW> keys(a, b, kh, first, count, tid, k_tile[side][0], v_tile[side][0]);
  if (WINDOW) keys.span = span_of(a, q0, held);
  const int tiles = keys.tiles(), steps = SIDES == 1 ? tiles : (tiles + SIDES - 1) / SIDES;
  v4i now, next;  // first keys of each sixteen of this tile and the next
  v16f acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = v16f{};
  const float c = a.scale * kLog2e;

  if (tid < 2) bad_tile[side][tid] = 0;
  if (a.dim < DP) {  // what no row fills stays zero
    for (int i = threadIdx.x; i < SIDES * 2 * KT * PIECES; i += 64 * NW * SIDES) ((v4i *)k_tile)[i] = ((v4i *)v_tile)[i] = v4i{0, 0, 0, 0};
    __syncthreads();
  }
  int ahead = 0;
  if (tiles > 0) {
    ahead = keys.look_up(SIDES + side);
    next = keys.spread(keys.look_up(side));
    keys.template load<0>(next);
  }
  lds_loads_done();
  __syncthreads();
  const auto step = [&](int t, auto which) {
    constexpr int buffer = decltype(which)::value;  // t & 1, known where addresses are made
    now = next;
    if (t + 1 < steps) {
      next = keys.spread(ahead);
      ahead = keys.look_up(SIDES * (t + 2) + side);
      keys.template load<1 - buffer>(next);
    }
    int lowest = now[0], top = now[0];
#pragma unroll
    for (int i = 1; i < CH; ++i) lowest = min(lowest, now[i]), top = max(top, now[i]);
    const bool cuts = top + 15 > low_of_all || (WINDOW && lowest <= gone_any_of_all);
    if (cuts) {  // somebody's mask cuts this tile: 0 times an infinity or NaN must not count
      bool bad = false;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) bad |= not_finite<T>(*(const vec8<T> *)(k_tile[side][buffer] + (p * NW * 64 + tid) * 8));
      if (__any(bad) && lane == 0) bad_tile[side][buffer] = t + 1;
      if (SIDES == 1) __syncthreads();
    }
    if (SIDES > 1) __syncthreads();  // of all, as one side's tile may be cut and not the other's
    if (lowest <= high) {
      const elem *kt = k_tile[side][buffer], *vt = v_tile[side][buffer];
      const bool cut = top + 15 > low || (WINDOW && lowest <= gone_any);
      const bool bad = cut && bad_tile[side][buffer] == t + 1;
      int place_lane = lane;  // made anew for each tile, or the compiler keeps the places of all operands in registers
      asm volatile("" : "+v"(place_lane));
#pragma unroll
      for (int x = 0; x < ST; ++x) {
        if (DP <= 64) asm volatile("" : "+v"(place_lane));  // or for each half of it: three wavefronts a SIMD
        // two chains of products that do not wait for each other, their operands read two products ahead
        constexpr int N = DP / 16, AHEAD = 2;
        v16f s = {}, g = {};
        vec8<T> ka[N], va[N];
        const auto read = [&](int y) {
          const int at = place_of<DP>(32 * x + (place_lane & 31), 2 * y + (place_lane >> 5));
          ka[y] = *(const vec8<T> *)(kt + at);
          va[y] = *(const vec8<T> *)(vt + at);
        };
#pragma unroll
        for (int y = 0; y < AHEAD; ++y) read(y);
        const auto score = [&](int y) {
          if (y + AHEAD < N) read(y + AHEAD);
          s = mfma32(ka[y], qf[y], s);
          g = mfma32(va[y], gf[y], g);
          __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int y = 0; y < N * 3 / 4; ++y) score(y);
        if (DP <= 64 || a.dim > 96) {  // the last quarter of a row, if it is there
#pragma unroll
          for (int y = N * 3 / 4; y < N; ++y) score(y);
        }
        // keys by columns for dQ, read some products ahead, the first of them before the exponentials
        vec8<T> kc[2 * DT], df[2];
        constexpr int LAST = DP <= 64 ? 0 : 2, FIRST = 2 * DT - LAST;  // products of the last 32 columns come last
        const auto key_of = [](int n) { return n < FIRST ? n / (FIRST / 2) : n - FIRST; };
        const auto column_of = [](int n) { return n < FIRST ? n % (FIRST / 2) : DT - 1; };
        const auto read_columns = [&](int n) { kc[n] = columns_in_order<T, DP>(kt, 32 * x + 16 * key_of(n), 32 * column_of(n), place_lane); };
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) read_columns(n);
        // dS is rounded to the operands' type for the product, with `scale` in it: smaller by its factor in float16's range
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -off)) * __builtin_fmaf(g[e], a.scale, -del);
        if (cut) {
          asm volatile("");  // (one branch, not one for each element)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = now[2 * x + (e >> 3)] + 8 * ((e >> 2) & 1) + 4 * half + (e & 3);
            s[e] = row_sees.sees(key) ? s[e] : 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) df[e >> 3][e & 7] = (elem)s[e];
        // a key's elements that are no numbers count for the rows that see it, by themselves; the product takes them as zeros
        int clean = !bad;  // either way, but not as two sides of one branch: the sums would be kept twice
        if (clean) {
          const auto product = [&](int n) {
            if (n + AHEAD < 2 * DT) read_columns(n + AHEAD);
            acc[column_of(n)] = mfma32(kc[n], df[key_of(n)], acc[column_of(n)]);
            __builtin_amdgcn_sched_barrier(0);
          };
#pragma unroll
          for (int n = 0; n < FIRST; ++n) product(n);
          if (LAST && a.dim > 96) {
#pragma unroll
            for (int n = FIRST; n < 2 * DT; ++n) product(n);
          }
        }
        asm volatile("" : "+v"(clean));
        if (__builtin_amdgcn_readfirstlane(clean) == 0) {
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < DT; ++i)
              acc[i] = mfma32(finite_only<T>(columns_in_order<T, DP>(kt, 32 * x + 16 * y, 32 * i, place_lane)), df[y], acc[i]);
#pragma unroll 1
          for (int row = 0; row < 32; ++row) {
            const int key = (row < 16 ? now[2 * x] : now[2 * x + 1]) + (row & 15);
            const bool sees = row_sees.sees(key);
            const float w = of_row<T>(df, row, lane);
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                const vec4<T> k = *(const vec4<T> *)(kt + place_of<DP>(32 * x + row, 4 * i + (e >> 2)) + 4 * half);
#pragma unroll
                for (int n = 0; n < 4; ++n)
                  if (sees && abs_bits((float)k[n]) >= kInfBits) acc[i][e + n] += w * (float)k[n];
              }
          }
        }
      }
    }
    lds_loads_done();
    __syncthreads();
  };
  for (int t = 0; t < steps; t += 2) {
    step(t, std::integral_constant<int, 0>());
    if (t + 1 < steps) step(t + 1, std::integral_constant<int, 1>());
  }
  if constexpr (SIDES > 1) {  // (the last step has ended with a barrier)
    float *sums = (float *)k_tile + wave * (DT * 1024) + lane * 4;
    if (side) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) *(v4f *)(sums + (4 * i + e / 4) * 256) = v4f{acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]};
    }
    __syncthreads();
    if (side) return;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] += sums[(4 * i + e / 4) * 256 + e % 4];
  }
  if (!live) return;
  elem *dp = (elem *)a.dq.data + b * a.dq.stride[0] + query * a.dq.stride[1] + head * a.dq.stride[2];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * i + 2 * e + 4 * half;
      vec4<T> x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (elem)acc[i][e + j];
      if (d < a.dim) *(vec4<T> *)(dp + d) = x;
    }
}

// Lists of few rows, as in the forward pass: 16 rows a wavefront, K and V from memory into the operands' registers, K through LDS
// for the product by columns.  SPLIT wavefronts share the keys of one list and add up, in their order, through LDS.
template <typename T, int DP, int SPLIT, bool WINDOW>
__global__ __launch_bounds__(256, DP <= 64 ? 4 : 2) void block_dq_narrow_kernel(BlockArgs a, int tiles_of_list, float *__restrict__ delta,
                                                                               float *__restrict__ logs, int *odd) {
  typedef typename T::elem elem;
  constexpr int KS = DP / 32, DT = DP / 16, PIECES = DP / 8;
  union Own {  // of a wavefront
    elem k[32 * DP];
    float out[16][DP + 4];
  };
  __shared__ __attribute__((aligned(16))) Own own[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quarter = lane >> 4;
  if (!WINDOW && blockIdx.x == 0 && tid <= kParts) odd[tid] = 0;  // for the kernels after this one: the flag and the counters behind it
  const int block = (int)(xcd_contiguous_block(blockIdx.x, gridDim.x) * (4 / SPLIT)) + wave / SPLIT, share = wave % SPLIT;
  const int list = block / tiles_of_list, part = block - list * tiles_of_list;
  const bool any = list < a.batch * a.kv_heads * a.rows;
  if (SPLIT == 1 && !any) return;  // no barrier below then
  const int bh = any ? list / a.rows : 0, r = any ? list - bh * a.rows : 0, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const int q0 = r * a.block_m, rows = min(a.block_m, a.queries - q0) * a.group;
  int first = 0, count = 0;
  Span span = {};
  if (any && part * 16 < rows) {
    if constexpr (WINDOW) span = span_of(a, q0, min(a.block_m, a.queries - q0));
    else entries_of(a, list, &first, &count);
  }
  const int row0 = part * 16, row = row0 + col, row_last = min(row0 + 15, rows - 1);
  const bool live = any && row < rows;
  const int query = q0 + row / a.group, head = kh * a.group + row % a.group;
  const int limit = a.causal ? min(query + a.shift, a.keys - 1) : a.keys - 1;
  const int low = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row0 / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int high = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row_last / a.group + a.shift, a.keys - 1) : a.keys - 1);

  vec8<T> qf[KS], gf[KS];
  float off = INFINITY, del = 0.f;  // of a row without entries: weights 0
  const elem *qp = (const elem *)a.q.data + b * a.q.stride[0] + query * a.q.stride[1] + head * a.q.stride[2];
  const elem *gp = (const elem *)a.dout.data + b * a.dout.stride[0] + query * a.dout.stride[1] + head * a.dout.stride[2];
  const elem *op = (const elem *)a.out.data + b * a.out.stride[0] + query * a.out.stride[1] + head * a.out.stride[2];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 32 * s + 8 * quarter;
    vec8<T> o = {};
    qf[s] = gf[s] = vec8<T>{};
    if (live && d < a.dim) {
      qf[s] = *(const vec8<T> *)(qp + d);
      gf[s] = *(const vec8<T> *)(gp + d);
      o = *(const vec8<T> *)(op + d);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) del += (float)gf[s][j] * (float)o[j];
  }
  del = rows_sum(del) * a.scale;
  if (live) {
    const long long at = ((long long)b * a.heads + head) * a.queries + query;
    const float lse = a.lse[at];
    off = lse == -INFINITY ? INFINITY : lse * kLog2e;
    if (quarter == 0 && share == 0) delta[at] = del, logs[at] = off;
  }
  const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + kh * a.k.stride[2];
  const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + kh * a.v.stride[2];
  const Sight<WINDOW> row_sees(a, limit);
  const int gone_any = high - a.window;  // last key before any row's window
  const int tiles = WINDOW ? (span.count + 1) / 2 : tiles_of<32>(a, count);
  v4i kr[2][KS], vr[2][KS];
  const auto load = [&](int key0, int key1) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int from = min(i ? key1 : key0, a.keys - 1), in = min(col, a.keys - 1 - from);
      const elem *k = kp + from * a.k.stride[1] + in * a.k.stride[1], *v = vp + from * a.v.stride[1] + in * a.v.stride[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 32 * s + 8 * quarter;
        kr[i][s] = *(const v4i *)(k + (d < a.dim ? d : 0));
        vr[i][s] = *(const v4i *)(v + (d < a.dim ? d : 0));
        if (a.dim < 32 * s + 32 && d >= a.dim) kr[i][s] = vr[i][s] = v4i{0, 0, 0, 0};
      }
    }
  };
  const auto look_up = [&](int t) {
    if constexpr (WINDOW) return span.first_key(2 * t + (lane & 1));
    return tiles > 0 ? first_key(a, first, count, 32ll * t + 16 * (lane & 1)) : kAbsent;
  };

  v4f acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  const float c = a.scale * kLog2e;
  elem *mine = own[wave].k;
  int ahead = look_up(share), next0 = __builtin_amdgcn_readlane(ahead, 0), next1 = __builtin_amdgcn_readlane(ahead, 1);
  if (share < tiles) load(next0, next1);
  ahead = look_up(share + SPLIT);
  for (int t = share; t < tiles; t += SPLIT) {
    const int now0 = next0, now1 = next1;
    v4f s[2], g[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = g[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        s[i] = mfma16(__builtin_bit_cast(vec8<T>, kr[i][x]), qf[x], s[i]);
        g[i] = mfma16(__builtin_bit_cast(vec8<T>, vr[i][x]), gf[x], g[i]);
      }
    }
    const bool cut = max(now0, now1) + 15 > low || (WINDOW && min(now0, now1) <= gone_any), skip = min(now0, now1) > high;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const int at = 16 * i + col, piece = 4 * x + quarter;
        if (cut) bad |= not_finite<T>(__builtin_bit_cast(vec8<T>, kr[i][x]));  // 0 times an infinity or NaN must not count
        *(v4i *)(mine + at * DP + ((piece ^ turn16<DP>(at)) * 8)) = kr[i][x];
      }
    bad = cut && __any(bad);
    next0 = __builtin_amdgcn_readlane(ahead, 0), next1 = __builtin_amdgcn_readlane(ahead, 1);
    if (t + SPLIT < tiles) load(next0, next1);
    ahead = look_up(t + 2 * SPLIT);
    if (skip) continue;
    vec8<T> df, kc[DT];
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < DT; ++i) {  // asked for before the exponentials
      const int x = 4 * quarter + (col >> 2), d = 16 * i + 4 * (col & 3);
      const elem *p = mine + x * DP + ((d >> 3) ^ turn16<DP>(x)) * 8 + (d & 7);  // row + 16 has the same order of pieces
      kc[i] = join<T>(read_columns<T>(p), read_columns<T>(p + 16 * DP));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], c, -off)) * __builtin_fmaf(g[i][e], a.scale, -del);
    if (cut) {
      asm volatile("");  // (one branch, not one for each element)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = row_sees.sees((i ? now1 : now0) + 4 * quarter + e) ? s[i][e] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) df[4 * i + e] = (elem)s[i][e];
    if (bad) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < DT; ++i) kc[i] = finite_only<T>(kc[i]);
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = mfma16(kc[i], df, acc[i]);
    if (bad)  // a key's elements that are no numbers, for the rows that see it
#pragma unroll 1
      for (int x = 0; x < 32; ++x) {
        const int key = (x < 16 ? now0 : now1) + (x & 15);
        const bool sees = row_sees.sees(key);
        float w = 0.f;  // key x is element 4 (x / 16) + x % 4 of quarter x / 4 % 4
#pragma unroll
        for (int e = 0; e < 8; ++e) w = e == 4 * (x >> 4) + (x & 3) ? (float)df[e] : w;
        w = __shfl(w, col | (x >> 2 & 3) << 4, 64);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const int d = 16 * i + 4 * quarter;
          const vec4<T> k = *(const vec4<T> *)(mine + x * DP + ((d >> 3) ^ turn16<DP>(x)) * 8 + (d & 7));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sees && abs_bits((float)k[e]) >= kInfBits) acc[i][e] += w * (float)k[e];
        }
      }
    wave_lds_sync();
  }
#pragma unroll
  for (int i = 0; i < DT; ++i) *(v4f *)(&own[wave].out[col][16 * i + 4 * quarter]) = acc[i];
  if (SPLIT == 1) wave_lds_sync();
  else __syncthreads();
  if (!any) return;
  const int w0 = SPLIT == 1 ? wave : 0;
  for (int x = SPLIT == 1 ? lane : tid; x < 16 * PIECES; x += SPLIT * 64) {
    const int h = x / PIECES, d = (x % PIECES) * 8;
    if (row0 + h >= rows || d >= a.dim) continue;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = own[w0].out[h][d + e];
#pragma unroll
    for (int w = 1; w < SPLIT; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += own[w0 + w].out[h][d + e];
    const int i = q0 + (row0 + h) / a.group, to = kh * a.group + (row0 + h) % a.group;
    *(vec8<T> *)((elem *)a.dq.data + b * a.dq.stride[0] + i * a.dq.stride[1] + to * a.dq.stride[2] + d) = narrow<T>(o);
  }
}

// ---- the columns' lists ----------------------------------------------------------------------------------------

// Which rows list a column, in ascending order (a row that lists it twice, twice).  Rows are cut into at most 64 chunks;
// counts[column][chunk], summed over a (batch entry, head)'s columns and chunks, gives each chunk its places.
struct Columns {
  int *odd;           // rows whose positions descend: with one of them rows overlap, and the lists are not made
  int *next;          // units taken from each part of them
  int *counts;        // lists x columns x chunks
  int *start, *end;   // of each column's rows; with positions that descend, end < 0: they were not found
  int *unit;          // column of each unit of work, -1 = nothing to do
  int *rows;          // nnz
  float *partial;     // of columns of several units: dk and dv of each
  int chunks, chunk_rows, per_unit, units, lists, sub;
};

__global__ void clear_kernel(int *p) { p[threadIdx.x] = 0; }

constexpr int kColumnsInLds = 8192, kRowsAtOnce = 16;

__device__ __forceinline__ long long position(const BlockArgs &a, long long row) { return min(max((long long)a.pos[row], 0ll), a.nnz); }

// One wavefront per chunk takes its rows one after the other, so that the places of a column ascend with its rows; the
// entries of sixteen rows are on their way at a time.
template <bool FILL>
__global__ __launch_bounds__(64) void columns_kernel(BlockArgs a, Columns t) {
  __shared__ int place[kColumnsInLds];
  if (FILL && *t.odd) return;
  const int lane = threadIdx.x, chunk = blockIdx.x, bh = blockIdx.z;
  const int c0 = blockIdx.y * kColumnsInLds, cs = min(kColumnsInLds, a.columns - c0);
  for (int c = lane; c < cs; c += 64) place[c] = FILL ? t.counts[((long long)bh * a.columns + c0 + c) * t.chunks + chunk] : 0;
  __syncthreads();
  const int r_end = min(a.rows, (chunk + 1) * t.chunk_rows);
  int odd = 0;
  const auto add = [&](int c, int r) {
    if ((unsigned)c < (unsigned)a.columns && c >= c0 && c < c0 + cs) {
      const int at = atomicAdd(&place[c - c0], 1);
      if (FILL && (unsigned)at < (unsigned long long)a.nnz) t.rows[at] = r;
    }
  };
  for (int r0 = chunk * t.chunk_rows; r0 < r_end; r0 += kRowsAtOnce) {
    int first = 0, count = 0, entry[kRowsAtOnce];
    bool descends = false;
    if (lane < kRowsAtOnce && r0 + lane < r_end) {
      const long long row = (long long)bh * a.rows + r0 + lane;
      entries_of(a, row, &first, &count);
      descends = position(a, row + 1) < first;
    }
    odd += __popcll(__ballot(descends));
    if (odd) continue;  // rows that overlap may name more entries than 32 bits count
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int f = __builtin_amdgcn_readlane(first, i), n = __builtin_amdgcn_readlane(count, i);
      entry[i] = lane < n ? a.crd[f + lane] : -1;
    }
#pragma unroll
    for (int i = 0; i < kRowsAtOnce; ++i) {
      const int f = __builtin_amdgcn_readlane(first, i), n = __builtin_amdgcn_readlane(count, i);
      add(entry[i], r0 + i);
      wave_lds_sync();
      for (int e = 64 + lane; e - lane < n; e += 64) {
        add(e < n ? a.crd[f + e] : -1, r0 + i);
        wave_lds_sync();
      }
    }
  }
  if (FILL) return;
  if (odd && lane == 0 && c0 == 0) atomicAdd(t.odd, odd);
  __syncthreads();
  for (int c = lane; c < cs; c += 64) t.counts[((long long)bh * a.columns + c0 + c) * t.chunks + chunk] = place[c];
}

// The units of work of a column: the places start / per_unit + column leave each column at least as many as it needs, so they
// are known without a sum over the columns before.  `next`: where the entries of the column after it start.
__device__ __forceinline__ void put_units(const Columns &t, int cc, int start, int rows, int next, bool last) {
  const int needed = max(1, (rows + t.per_unit - 1) / t.per_unit);
  const long long to = (long long)start / t.per_unit + cc, stop = last ? t.units : (long long)next / t.per_unit + cc + 1;
  for (long long u = to; u < stop && u < t.units; ++u) t.unit[u] = u < to + needed ? cc : -1;
  if (cc == 0)  // positions may start past 0
    for (long long u = 0; u < to && u < t.units; ++u) t.unit[u] = -1;
}

// Where a list's entries start (positions are in order here).
__device__ __forceinline__ int list_start(const BlockArgs &a, long long bh) { return a.rows ? (int)position(a, bh * a.rows) : 0; }

// One workgroup per (batch entry, key-value head): counts become places, columns get their ranges and their units of work.
__global__ __launch_bounds__(1024) void columns_scan_kernel(BlockArgs a, Columns t) {
  __shared__ int wave_sum[16], total;
  if (*t.odd) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bh = blockIdx.x;
  if (tid == 0) total = list_start(a, bh);
  const long long n = (long long)a.columns * t.chunks;
  int *counts = t.counts + bh * n;
  __syncthreads();
  for (long long i0 = 0; i0 < n; i0 += 4096) {
    int v[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = i0 + tid * 4 + j;
      v[j] = i < n ? counts[i] : 0;
      sum += v[j];
    }
    int upto = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    int before = total;
    for (int w = 0; w < wave; ++w) before += wave_sum[w];
    int at = before + upto - sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = i0 + tid * 4 + j;
      if (i < n) {
        counts[i] = at;
        if (i % t.chunks == 0) t.start[bh * (long long)a.columns + i / t.chunks] = at;
      }
      at += v[j];
      if (i < n && i % t.chunks == t.chunks - 1) t.end[bh * (long long)a.columns + i / t.chunks] = at;
    }
    __syncthreads();
    if (tid == 1023) total = at;
    __syncthreads();
  }
  __threadfence_block();
  __syncthreads();
  for (int c = tid; c < a.columns; c += 1024) {
    const int cc = bh * a.columns + c, start = t.start[cc], end = t.end[cc];
    put_units(t, cc, start, end - start, c + 1 < a.columns ? end : list_start(a, bh + 1ll), c + 1 == a.columns && bh + 1 == t.lists);
  }
}

// All of it in one workgroup per (batch entry, key-value head) where rows and columns are few: a chunk of rows to each of its
// wavefronts, the counts in LDS.  (Three launches less two: 14 us become 6 at 128 rows and columns.)
constexpr int kFewColumns = 1024, kFewRows = 512;
__global__ __launch_bounds__(1024) void few_columns_kernel(BlockArgs a, Columns t) {
  __shared__ int place[kFewColumns * 16];  // [column][wavefront]
  __shared__ int wave_sum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bh = blockIdx.x;
  const int rows_each = (a.rows + 15) / 16, r0 = wave * rows_each, r1 = min(a.rows, r0 + rows_each);  // at most 32
  for (int i = tid; i < a.columns * 16; i += 1024) place[i] = 0;
  int first = 0, count = 0;
  bool odd = false;
  if (lane < rows_each && r0 + lane < r1) {
    const long long row = (long long)bh * a.rows + r0 + lane;
    entries_of(a, row, &first, &count);
    odd = position(a, row + 1) < first;
  }
  const int descents = __popcll(__ballot(odd));
  if (descents && lane == 0) atomicAdd(t.odd, descents);
  if (lane == 0) wave_sum[wave] = descents;
  __syncthreads();
  int of_list = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) of_list |= wave_sum[w];
  if (of_list) return;
  const auto pass = [&](bool fill) {  // a wavefront's rows one after the other, their first entries asked for eight at a time
    for (int i0 = 0; i0 < r1 - r0; i0 += 8) {
      int entry[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int f = __builtin_amdgcn_readlane(first, (i0 + i) & 63), n = i0 + i < r1 - r0 ? __builtin_amdgcn_readlane(count, (i0 + i) & 63) : 0;
        entry[i] = lane < n ? a.crd[f + lane] : -1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int f = __builtin_amdgcn_readlane(first, (i0 + i) & 63), n = i0 + i < r1 - r0 ? __builtin_amdgcn_readlane(count, (i0 + i) & 63) : 0;
        for (int e = lane; e - lane < n; e += 64) {
          const int c = e < 64 ? entry[i] : e < n ? a.crd[f + e] : -1;
          if ((unsigned)c < (unsigned)a.columns) {
            const int at = atomicAdd(&place[c * 16 + wave], 1);
            if (fill && (unsigned)at < (unsigned long long)a.nnz) t.rows[at] = r0 + i0 + i;
          }
          wave_lds_sync();
        }
      }
    }
  };
  pass(false);
  __syncthreads();
  // a column to a thread: its sixteen counts, and the sum over the columns before
  int sum = 0;
  if (tid < a.columns)
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += place[tid * 16 + w];
  int upto = sum;
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o, 64);
    if (lane >= o) upto += x;
  }
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  int start = list_start(a, bh) + upto - sum;
  for (int w = 0; w < wave; ++w) start += wave_sum[w];
  if (tid < a.columns) {
    int at = start;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const int n = place[tid * 16 + w];
      place[tid * 16 + w] = at;
      at += n;
    }
    const int cc = bh * a.columns + tid;
    t.start[cc] = start;
    t.end[cc] = at;
    put_units(t, cc, start, sum, tid + 1 < a.columns ? at : list_start(a, bh + 1ll), tid + 1 == a.columns && bh + 1 == t.lists);
  }
  __syncthreads();
  pass(true);
}

// ---- dK and dV -------------------------------------------------------------------------------------------------

constexpr int kMostEntries = 384;  // of a unit
constexpr int kMostDescents = 16;  // of positions: 17 times the entries at most

// A unit of work: 32 * KG keys of a column and some of the rows that list it, their queries times heads packed into tiles of
// 32.  Two wavefronts share 32 keys, a key per lane, K and V of them in registers: one computes S and P (queries x keys), which
// feeds dV^T = dO^T P from its registers; the other S, P, dP and dS, which feeds dK^T = Q^T dS.  Both sums in one wavefront take
// 318 registers, one wavefront a SIMD and nothing to fill the waits with (1.06 ms at 8k queries); P handed over
// through LDS saves a product of five, but its barrier in the middle of every tile costs more (0.67 ms against 0.57).
// Where keys are few (KG = 1) two pairs take turns with the tiles and add up at the end.
// An iteration turns the scores of its tile into weights, then multiplies by them and computes the scores of the next tile in
// turn, three chains of products that do not wait for each other; where the rows of four tiles lie is worked out by 128
// threads at once, and what an iteration needs from LDS is asked for a stage before its use.  (A single workgroup, 64 keys,
// dim 128: 1.35 us an iteration with one chain after the other, 1.10 so; 8192 queries, 32 heads over 8, 16 blocks of 64
// a row: 630 us to 549, in a trace; 511 now.)  It is bound by what an iteration of a wavefront waits for: the products alone are 128 us.
// The rows of a column lie all over Q and dO, beyond L2 in large passes (16 columns read each block of rows: 2.1 GB, 290 us
// by themselves): S tiles are on their way or being computed, and no load but those into LDS is in the loop.
// Columns are anything but equal (the first block is listed by all rows, the last by few): workgroups take units from a
// counter, those of their XCD's part first, whose rows of Q and dO its L2 holds.
// The kernel's arguments are more than the scalar registers hold beside the loop (148 spilled, and a wait for a spilled register in
// the loop waits for the tiles on their way too), so whatever the loop does not need all the time is read from the arguments
// again where it is used (at dim 128, 64 keys, about 50 spilled, and 13 vector registers, none in the loop over tiles).
struct DkvArgs {
  BlockArgs a;
  Columns cols;
  const float *delta, *logs;
};
typedef const __attribute__((address_space(4))) DkvArgs *DkvArgsAgain;
__device__ __forceinline__ DkvArgsAgain again() {
  DkvArgsAgain p = (DkvArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// What all lanes of a wavefront agree on, said so that the compiler branches on it and does not walk through both sides.
__device__ __forceinline__ bool same(bool x) { return __builtin_amdgcn_readfirstlane((int)x) != 0; }

// Where positions descend rows overlap and there are no lists of columns: the rows that name column cc (counted through all lists)
// are looked for, by a workgroup of 256.  Rows whose positions ascend hold neighbouring entries, which are compared 256 at a time; each
// descent may bring all entries once more.  Returns how many there are, in order, in `rows`; -1: more than that holds, or
// descents without end.
__device__ __forceinline__ int rows_that_name(const BlockArgs &a, int cc, int descents, int *rows, int *found) {
  if (descents > kMostDescents) return -1;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bh = cc / a.columns, column = cc - bh * a.columns;
  const long long row0 = (long long)bh * a.rows;
  const auto threads_that = [&](bool x, int *before) {  // say so, and how many of them come before this one
    const unsigned long long these = __ballot(x);
    __syncthreads();
    if (lane == 0) found[wave] = __popcll(these);
    __syncthreads();
    int all = 0;
    *before = __popcll(these & ((1ull << lane) - 1));
    for (int w = 0; w < 4; ++w) {
      if (w < wave) *before += found[w];
      all += found[w];
    }
    return __builtin_amdgcn_readfirstlane(all);
  };
  int n = 0, before;
  for (int r0 = 0, r1; r0 < a.rows; r0 = r1) {
    r1 = min(r0 + 256, a.rows);
    const long long r = row0 + min(r0 + tid, r1 - 1);
    if (threads_that(position(a, r + 1) < position(a, r), &before) > 0) r1 = r0 + 1;
    const long long end = position(a, row0 + r1);
    for (long long e0 = position(a, row0 + r0); e0 < end; e0 += 256) {
      const long long e = e0 + tid;
      const bool names = e < end && a.crd[e] == column;
      const int more = threads_that(names, &before);
      if (n + more > kMostEntries) return -1;
      if (names) {
        int lo = r0, hi = r1;  // row lo starts at or before entry e, row hi behind it
        while (hi - lo > 1) {
          const int middle = lo + (hi - lo) / 2;
          if (position(a, row0 + middle) <= e) lo = middle;
          else hi = middle;
        }
        rows[n + before] = lo;
      }
      n += more;
    }
  }
  return n;
}

template <typename T, int DP, int KG, int S>
struct DkvShared {
  static constexpr int QG = 2 / KG, BATCH = 4;
  struct Info {  // where a tile's rows lie
    long long q[32], g[32];
    int sums[32], last[32];
  };
  __attribute__((aligned(16))) typename T::elem tiles[QG][S][2][32 * DP];
  __attribute__((aligned(16))) float sums[QG][S][2][32];  // log-sums and deltas of a tile's rows
  __attribute__((aligned(16))) Info infos[QG][2 * BATCH];
  int rows_of_unit[kMostEntries], taken, found[4];
};

// ODD: positions descend.  A body of its own, as the kernel's own look for rows among its units costs the loop registers (8192 queries, 16
// blocks of 64: 547 us against 510).
template <typename T, int DP, int KG, int S, bool ODD>
__device__ __forceinline__ void dkv_units(const DkvArgs &args, DkvShared<T, DP, KG, S> &mem) {
  typedef typename T::elem elem;
  typedef typename DkvShared<T, DP, KG, S>::Info Info;
  constexpr int QG = 2 / KG, TG = KG * 128, PIECES = DP / 8, RP = TG / PIECES, PASSES = 32 / RP, DT = DP / 32, BATCH = 4;
  static_assert(S <= BATCH, "what is loaded is looked up a batch before");
  auto &tiles = mem.tiles;
  auto &sums = mem.sums;
  auto &infos = mem.infos;
  auto &rows_of_unit = mem.rows_of_unit;
  int &taken = mem.taken;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int role = (wave ^ blockIdx.x / kParts) & 1, kg = (wave >> 1) % KG, qg = (wave >> 1) / KG, gt = tid - qg * TG;  // role 0: dV, 1: dK
  const int all_units = (ODD ? args.cols.lists * args.a.columns : args.cols.units) * args.cols.sub;
  const float scale = args.a.scale, c = scale * kLog2e;
  const int dim = args.a.dim;
  const elem *const all_q = (const elem *)args.a.q.data, *const all_g = (const elem *)args.a.dout.data;

  // One unit for each workgroup, or units from the counters: those of the own part, then of whichever part has some left.
  const bool one_each = all_units <= (int)gridDim.x;
  const auto part_start = [&](int p) { return (int)((long long)all_units * p / kParts); };
  int part = blockIdx.x % kParts;
  for (bool more = true; more;) {
    int unit_l;
    if (one_each) {
      unit_l = (int)xcd_contiguous_block(blockIdx.x, gridDim.x);
      if (unit_l >= all_units) return;
      more = false;
    } else {
      __syncthreads();
      int *const next = again()->cols.next;
      if (tid == 0) taken = atomicAdd(next + part, 1);
      __syncthreads();
      unit_l = part_start(part) + taken;
      if (unit_l >= part_start(part + 1)) {
        bool left = false;
        if (lane < kParts) {
          const int p = (part + lane) % kParts;
          left = part_start(p) + __hip_atomic_load(next + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) < part_start(p + 1);
        }
        __syncthreads();
        if (wave == 0) {
          const unsigned long long some = __ballot(left);
          if (lane == 0) taken = some ? (part + __ffsll((long long)some) - 1) % kParts : -1;
        }
        __syncthreads();
        part = taken;
        more = part >= 0;
        continue;
      }
    }
    const DkvArgsAgain at_start = again();
    const auto &a = at_start->a;
    const auto &cols = at_start->cols;
    const int u = unit_l / cols.sub, sub = unit_l - u * cols.sub;
    int cc, from = 0, n = 0, start = 0;
    bool several = false;
    if (ODD) {
      cc = u;
      n = rows_that_name(*(const BlockArgs *)&at_start->a, cc, *cols.odd, rows_of_unit, mem.found);
      if (tid == 0) cols.end[cc] = n;
      if (n < 0) continue;  // NaN: the next kernel
    } else {
      cc = cols.unit[u];
      if (cc < 0) continue;
      start = cols.start[cc];
      const int rows = cols.end[cc] - start;
      several = rows > cols.per_unit;
      from = (u - (start / cols.per_unit + cc)) * cols.per_unit;
      n = min(rows - from, cols.per_unit);
      for (int e = tid; e < n; e += 256) rows_of_unit[e] = cols.rows[start + from + e];
    }
    const int bh = cc / a.columns, column = cc - bh * a.columns, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
    const int in_block = sub * 32 * KG + kg * 32;
    const int key_low = (column << a.block_n_log2) + in_block, key = key_low + (lane & 31);
    const bool live = in_block + (lane & 31) < (1 << a.block_n_log2) && key < a.keys;

    // Where rows lie is worked out for four tiles of a group at a time, a row to each of 128 threads: one wavefront doing it in
    // every iteration is what all others wait for.  A thread's row: entry, query of the block and head of the group.
    const int looks_up = KG == 2 ? (role ? 128 : kg * 64 + lane) : gt, steps = BATCH * 32 * QG;
    const int steps_h = steps % a.group, steps_q = steps / a.group % a.block_m, steps_e = steps / a.group / a.block_m;
    const int slot0 = ((looks_up >> 5) * QG + qg) * 32 + (looks_up & 31);
    int entry = slot0 / a.group / a.block_m, in = slot0 / a.group % a.block_m, hd = slot0 % a.group;
    const long long all = (long long)n * a.block_m * a.group;
    const int tiles_n = (int)((all + 32 * QG - 1) / (32 * QG));
    const auto put_info = [&](int t) {  // of tiles t .. t + 3, batches in turn
      if (looks_up >= 128) return;
      const auto &a = again()->a;
      {
        Info &i = infos[qg][(t + (looks_up >> 5)) % (2 * BATCH)];
        const int lane = looks_up & 31;
        int query = 0;
        bool there = entry < n;
        if (there) {
          query = rows_of_unit[entry] * a.block_m + in;
          there = query < a.queries;
        }
        query = there ? query : 0;
        const int head = kh * a.group + hd;
        i.q[lane] = b * a.q.stride[0] + query * a.q.stride[1] + head * a.q.stride[2];
        i.g[lane] = b * a.dout.stride[0] + query * a.dout.stride[1] + head * a.dout.stride[2];
        i.sums[lane] = (b * a.heads + head) * a.queries + query;
        i.last[lane] = !there ? -1 : a.causal ? min(query + a.shift, a.keys - 1) : a.keys - 1;
      }
      hd += steps_h;
      in += steps_q;
      entry += steps_e;
      if (hd >= a.group) hd -= a.group, ++in;
      if (in >= a.block_m) in -= a.block_m, ++entry;
    };
    const int place = gt % PIECES, my_row = gt / PIECES, in_group = wave - qg * KG * 2;
    constexpr int LOADS = 2 * PASSES;  // at least that many a tile and wavefront
    struct Places {  // of what this thread loads of a tile
      long long q[PASSES], g[PASSES];
      int sums;
    };
    const auto look = [&](int t) {
      const Info &i = infos[qg][t % (2 * BATCH)];
      Places at;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) at.q[p] = i.q[p * RP + my_row], at.g[p] = i.g[p * RP + my_row];
      at.sums = i.sums[lane & 31];
      return at;
    };
    const auto load = [&](int t, const Places &from) {
      const int slot = t % S;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int d = (place ^ turn<DP>(p * RP + my_row)) * 8;
        const unsigned to = __builtin_amdgcn_readfirstlane(lds_address(tiles[qg][slot][0]) + (p * KG * 2 + in_group) * 1024);
        if (d < dim) {
          load_to_lds(all_q + from.q[p] + d, to);
          load_to_lds(all_g + from.g[p] + d, to + 64 * DP);
        }
      }
      if (role == 0 && kg == 0 && lane < 32) {
        const unsigned to = __builtin_amdgcn_readfirstlane(lds_address(sums[qg][slot][0]));
        load_word_to_lds(args.logs + from.sums, to);
        load_word_to_lds(args.delta + from.sums, to + 128);
      }
    };

    v16f acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = v16f{};
    // The two roles have a loop of their own each, the same barriers in both: what one of them keeps in registers is not kept
    // free in the other.
    const auto run = [&](auto with_g) {
      constexpr bool G = decltype(with_g)::value;
      vec8<T> kf[DP / 16], vf[DP / 16];
      const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + key * a.k.stride[1] + kh * a.k.stride[2];
      const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + key * a.v.stride[1] + kh * a.v.stride[2];
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        const int d = 16 * s + 8 * half;
        kf[s] = vf[s] = vec8<T>{};
        if (live && d < dim) kf[s] = *(const vec8<T> *)(kp + d);
        if (G && live && d < dim) vf[s] = *(const vec8<T> *)(vp + d);
      }

      if (dim < DP)  // what no row fills stays zero
        for (int i = tid; i < QG * S * 2 * 32 * PIECES; i += 256) ((v4i *)tiles)[i] = v4i{0, 0, 0, 0};
      __syncthreads();
      put_info(0);
      put_info(BATCH);
      __syncthreads();
      for (int t = 0; t < S - 1; ++t)
        if (t < tiles_n) load(t, look(t));
      lds_loads_done();
      __syncthreads();
      // An iteration turns the scores of its tile into weights, then multiplies by them and computes the next tile's scores: three
      // chains of products that do not wait for each other.
      int place_lane = lane;  // made anew in each iteration, or the compiler keeps the places of all operands in registers
      const auto rows_of = [&](const elem *tile, int y) { return *(const vec8<T> *)(tile + place_of<DP>(place_lane & 31, 2 * y + (place_lane >> 5))); };
      const auto last_of = [&](int t) { return infos[qg][t % (2 * BATCH)].last[lane & 31]; };
      v16f s = {}, g = {};
      int last = last_of(0);
      bool now = tiles_n > 0 && same(__any(last >= key_low));
      constexpr int N = DP / 16;
#pragma unroll
      for (int y = 0; y < N; ++y) s = mfma32(rows_of(tiles[qg][0][0], y), kf[y], s);
      if (G) {
#pragma unroll
        for (int y = 0; y < N; ++y) g = mfma32(rows_of(tiles[qg][0][1], y), vf[y], g);
      }
      for (int t = 0; t < tiles_n; ++t) {
        asm volatile("" : "+v"(place_lane));
        if (t % BATCH == 0 && t > 0 && t + BATCH < tiles_n) put_info(t + BATCH);
        // asked for here, used after the weights
        const int last_next = last_of(t + 1);
        const Places from = look(t + S - 1);
        const elem *qt = tiles[qg][(t + 1) % S][0], *dt = tiles[qg][(t + 1) % S][1], *by_column = tiles[qg][t % S][G ? 0 : 1];
        vec8<T> f[2] = {};
        unsigned bad = 0;
        if (now) {
          const Info &info = infos[qg][t % (2 * BATCH)];
          const bool cut = same(__any(last < key_low + 31));
          const float *lse = sums[qg][t % S][0], *dl = sums[qg][t % S][1];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v4f off = *(const v4f *)(lse + 8 * j + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * j + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * j + e], c, -off[e]));
          }
          if (G) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const v4f del = *(const v4f *)(dl + 8 * j + 4 * half);
#pragma unroll
              for (int e = 0; e < 4; ++e) s[4 * j + e] *= __builtin_fmaf(g[4 * j + e], scale, -del[e]);
            }
          }
          if (cut) {
            // 0 times an infinity or NaN must not count: which rows of the last product's operand hold one?
#pragma unroll 1
            for (int i = 0; i < PIECES / 2; ++i) {
              const unsigned long long lanes = __ballot(not_finite<T>(*(const vec8<T> *)(by_column + (i * 64 + lane) * 8)));
              if (lanes == 0) continue;
#pragma unroll
              for (int x = 0; x < 64 / PIECES; ++x)
                if (lanes >> (x * PIECES) & ((1u << PIECES) - 1)) bad |= 1u << (i * (64 / PIECES) + x);
            }
            bad = __builtin_amdgcn_readfirstlane(bad);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const v4i lim = *(const v4i *)(info.last + 8 * j + 4 * half);
#pragma unroll
              for (int e = 0; e < 4; ++e) s[4 * j + e] = key <= lim[e] ? s[4 * j + e] : 0.f;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e >> 3][e & 7] = (elem)s[e];
          // The operand's elements that are no numbers, for the keys that their rows see; the product below takes them as zeros.
#pragma unroll 1
          for (unsigned left = bad; left != 0; left &= left - 1) {
            const int row = __builtin_ctz(left);
            const float w = of_row<T>(f, row, lane);
            const bool sees = key <= infos[qg][t % (2 * BATCH)].last[row];
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                const vec4<T> x = *(const vec4<T> *)(by_column + place_of<DP>(row, 4 * i + (e >> 2)) + 4 * half);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                  const float y = (float)x[n];
                  if (sees && abs_bits(y) >= kInfBits) acc[i][e + n] += w * y;
                }
              }
          }
        }
        if (t + S - 1 < tiles_n) load(t + S - 1, from);
        const bool next = t + 1 < tiles_n && same(__any(last_next >= key_low));
        last = last_next;
        s = v16f{};
        g = v16f{};
        const auto column = [&](int y) { return columns_in_order<T, DP>(by_column, 16 * (y / DT), 32 * (y % DT), place_lane); };
        // Either of two ways through, but not as two sides of one branch: the sums would be kept twice.
        const bool fast = now && bad == 0;
        if (fast) {  // (scores of a tile that no row sees are not used)
          // operands are read some products ahead of their use: left to itself the compiler reads each one just before
          constexpr int AHEAD = 2;
          static_assert(2 * DT == N, "as many products of weights as of a score");
          vec8<T> qa[N], ga[N], x[N];
          const auto read = [&](int y) {
            qa[y] = rows_of(qt, y);
            if (G) ga[y] = rows_of(dt, y);
            x[y] = column(y);
          };
#pragma unroll
          for (int y = 0; y < AHEAD; ++y) read(y);
#pragma unroll
          for (int y = 0; y < N; ++y) {
            if (y + AHEAD < N) read(y + AHEAD);
            s = mfma32(qa[y], kf[y], s);
            if (G) g = mfma32(ga[y], vf[y], g);
            acc[y % DT] = mfma32(x[y], f[y / DT], acc[y % DT]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        int slow = !fast;
        asm volatile("" : "+v"(slow));
        if (__builtin_amdgcn_readfirstlane(slow)) {
          if (now) {
#pragma unroll
            for (int y = 0; y < N; ++y) acc[y % DT] = mfma32(finite_only<T>(column(y)), f[y / DT], acc[y % DT]);
          }
          if (next) {
#pragma unroll
            for (int y = 0; y < N; ++y) s = mfma32(rows_of(qt, y), kf[y], s);
            if (G) {
#pragma unroll
              for (int y = 0; y < N; ++y) g = mfma32(rows_of(dt, y), vf[y], g);
            }
          }
        }
        now = next;
        // the tile after the next one has to be there
        if (t + S - 1 < tiles_n) lds_loads_done<(S - 3) * LOADS>();
        else lds_loads_done();
        __syncthreads();
      }
    };
    if (role) run(std::true_type());
    else run(std::false_type());
    if (QG > 1) {  // the second pair's sums to the first, with the tiles' memory between them
      float *between = (float *)tiles + role * DT * 1024;
      if (qg > 0) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) between[(i * 16 + e) * 64 + lane] = acc[i][e];
      }
      __syncthreads();
      if (qg == 0) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][e] += between[(i * 16 + e) * 64 + lane];
      }
    }
    if (qg > 0 || !live) continue;
    const DkvArgsAgain at_end = again();
    if (several) {
      const auto &cols = at_end->cols;
      const long long slot = 2ll * (start / cols.per_unit) + from / cols.per_unit, each = (long long)DP << at_end->a.block_n_log2;
      float *to = cols.partial + (slot * 2 + 1 - role) * each + (long long)(in_block + (lane & 31)) * DP;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) *(v4f *)(to + 32 * i + 2 * e + 4 * half) = v4f{acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]};
      continue;
    }
    const auto &dkv = role ? at_end->a.dk : at_end->a.dv;
    elem *to = (elem *)dkv.data + b * dkv.stride[0] + key * dkv.stride[1] + kh * dkv.stride[2];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * i + 2 * e + 4 * half;
        vec4<T> x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (elem)acc[i][e + j];
        if (d < dim) *(vec4<T> *)(to + d) = x;
      }
  }
}

template <typename T, int DP, int KG, int S>
__global__ __launch_bounds__(256, 2) void block_dkv_kernel(DkvArgs args) {
  __shared__ DkvShared<T, DP, KG, S> mem;
  if (same(*args.cols.odd != 0)) dkv_units<T, DP, KG, S, true>(args, mem);
  else dkv_units<T, DP, KG, S, false>(args, mem);
}

// Columns of several units: their sums, in the order of the units.  NaN where the rows of a column were not found.
template <typename T, int DP>
__global__ __launch_bounds__(256) void join_units_kernel(BlockArgs a, Columns cols) {
  typedef typename T::elem elem;
  const int cc = blockIdx.x;
  const bool odd = *cols.odd != 0, lost = odd && cols.end[cc] < 0;
  const int start = odd ? 0 : cols.start[cc], rows = odd ? 0 : cols.end[cc] - start;
  if (rows <= cols.per_unit && !lost) return;
  const int units = (rows + cols.per_unit - 1) / cols.per_unit;
  const int bh = cc / a.columns, column = cc - bh * a.columns, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const long long each = (long long)DP << a.block_n_log2;
  const float *from = cols.partial + 2ll * (start / cols.per_unit) * 2 * each;
  for (long long x = (blockIdx.y * 256 + threadIdx.x) * 4; x < 2 * each; x += 4096) {
    const bool is_v = x >= each;
    const int at = (int)(is_v ? x - each : x), d = at % DP, key = (column << a.block_n_log2) + at / DP;
    if (key >= a.keys || d >= a.dim) continue;
    const float none = lost ? __builtin_nanf("") : 0.f;
    v4f sum = {none, none, none, none};
    for (int j = 0; j < units; ++j) {
      const v4f y = *(const v4f *)(from + j * 2 * each + x);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += y[e];
    }
    const View &v = is_v ? a.dv : a.dk;
    vec4<T> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (elem)sum[e];
    *(vec4<T> *)((elem *)v.data + b * v.stride[0] + key * v.stride[1] + kh * v.stride[2] + d) = o;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------

struct Layout {
  int64_t delta, logs, odd, counts, start, end, unit, rows, partial, bytes;
  Columns columns;
};

// How dQ is launched.
struct DqGrid {
  bool few, many;
  long long tiles, blocks;
};

DqGrid dq_grid(const BlockArgs &a) {
  const long long lists = (long long)a.batch * a.kv_heads * a.rows, rows = (long long)a.block_m * a.group;
  // the forward pass's rule: short lists, or few of them
  const bool few = rows <= 32 || ceil_div(rows, 128) * lists < device_cu_count() / 2, many = ceil_div(rows, 16) * lists >= 8 * device_cu_count();
  const long long tiles = ceil_div(rows, few ? 16 : 128);
  return {few, many, tiles, few ? ceil_div(lists * tiles * (many ? 1 : 4), 4) : lists * tiles};
}

int layout_of(const BlockArgs &a, Layout *layout) {
  const int64_t lists = (int64_t)a.batch * a.kv_heads, columns = lists * a.columns;
  LAPIS_REQUIRE(lists <= 65535 && columns * 256 < (INT64_C(1) << 32), "block_attention_backward: %lld lists of %d columns", (long long)lists, a.columns);
  LAPIS_REQUIRE(a.rows == 0 || dq_grid(a).blocks * 256 < (INT64_C(1) << 32), "block_attention_backward: %lld rows of the structure",
                (long long)lists * a.rows);
  Layout &l = *layout = {};
  Columns &c = l.columns;
  c.lists = a.batch * a.kv_heads;
  c.chunk_rows = (int)std::max<int64_t>(kRowsAtOnce, ceil_div(ceil_div(a.rows, 64), kRowsAtOnce) * kRowsAtOnce);
  c.chunks = (int)std::max<int64_t>(1, ceil_div(a.rows, c.chunk_rows));
  // Up to 8192 queries times heads a unit, so that long columns do not stand alone and those of ordinary length need no join; in
  // small passes what gives every workgroup one (the first block's column is all there is to wait for otherwise).
  const int64_t rows_of_entry = (int64_t)std::min(a.block_m, std::max(a.queries, 1)) * std::max(a.group, 1);
  const int64_t rows_of_unit = std::min<int64_t>(std::max<int64_t>(a.nnz * rows_of_entry / std::max(device_cu_count(), 1), 256), 8192);
  c.per_unit = (int)std::min<int64_t>(kMostEntries, std::max<int64_t>(1, rows_of_unit / rows_of_entry));
  const int64_t units = a.nnz / c.per_unit + columns;
  LAPIS_REQUIRE(units * 8 <= INT32_MAX, "block_attention_backward: %lld units of work", (long long)units);  // of up to eight parts each
  c.units = (int)units;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.delta = take(4ll * a.batch * a.heads * a.queries);
  l.logs = take(4ll * a.batch * a.heads * a.queries);
  l.odd = take(4 * (1 + kParts));
  l.counts = take(4ll * c.lists * a.columns * c.chunks);
  l.start = take(4ll * c.lists * a.columns);
  l.end = take(4ll * c.lists * a.columns);
  l.unit = take(4ll * c.units);
  l.rows = take(4 * a.nnz);
  const int dp = a.dim <= 64 ? 64 : 128;
  l.partial = take(2 * (a.nnz / c.per_unit) * 2 * ((int64_t)dp << a.block_n_log2) * 4);
  l.bytes = at;
  return LAPIS_HIP_OK;
}

template <typename T, int DP, int KG, int S>
void launch_dkv(const BlockArgs &a, const Columns &c, const float *delta, const float *logs, hipStream_t st) {
  Columns cols = c;
  cols.sub = (int)ceil_div(1 << a.block_n_log2, 32 * KG);
  const int64_t grid = std::min<int64_t>(2 * device_cu_count(), (int64_t)c.units * cols.sub);
  hipLaunchKernelGGL((block_dkv_kernel<T, DP, KG, S>), dim3((unsigned)grid), dim3(256), 0, st, DkvArgs{a, cols, delta, logs});
}

template <typename T, int DP>
int launch_backward(const BlockArgs &a, char *work, hipStream_t st) {
  Layout l;
  const int rc = layout_of(a, &l);
  if (rc != LAPIS_HIP_OK) return rc;
  Columns &c = l.columns;
  float *delta = reinterpret_cast<float *>(work + l.delta), *logs = reinterpret_cast<float *>(work + l.logs);
  c.odd = reinterpret_cast<int *>(work + l.odd);
  c.next = c.odd + 1;
  c.counts = reinterpret_cast<int *>(work + l.counts);
  c.start = reinterpret_cast<int *>(work + l.start);
  c.end = reinterpret_cast<int *>(work + l.end);
  c.unit = reinterpret_cast<int *>(work + l.unit);
  c.rows = reinterpret_cast<int *>(work + l.rows);
  c.partial = reinterpret_cast<float *>(work + l.partial);
  if (a.rows) {
    const DqGrid g = dq_grid(a);
    const auto kernel = !g.few ? block_dq_kernel<T, DP, 4, 64, false> : g.many ? block_dq_narrow_kernel<T, DP, 1, false> : block_dq_narrow_kernel<T, DP, 4, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)g.blocks), dim3(256), 0, st, a, (int)g.tiles, delta, logs, c.odd);
  }
  if (c.lists && a.columns) {
    if (a.rows == 0) hipLaunchKernelGGL(clear_kernel, dim3(1), dim3(1 + kParts), 0, st, c.odd);  // no dQ kernel has done it
    const dim3 grid((unsigned)c.chunks, (unsigned)ceil_div(a.columns, kColumnsInLds), (unsigned)c.lists);
    if (a.columns <= kFewColumns && a.rows <= kFewRows) {
      hipLaunchKernelGGL(few_columns_kernel, dim3((unsigned)c.lists), dim3(1024), 0, st, a, c);
    } else {
      hipLaunchKernelGGL(columns_kernel<false>, grid, dim3(64), 0, st, a, c);
      hipLaunchKernelGGL(columns_scan_kernel, dim3((unsigned)c.lists), dim3(1024), 0, st, a, c);
      hipLaunchKernelGGL(columns_kernel<true>, grid, dim3(64), 0, st, a, c);
    }
    if (a.block_n_log2 <= 5) launch_dkv<T, DP, 1, DP == 64 ? 4 : 3>(a, c, delta, logs, st);
    else launch_dkv<T, DP, 2, 4>(a, c, delta, logs, st);
    hipLaunchKernelGGL((join_units_kernel<T, DP>), dim3((unsigned)(c.lists * a.columns), 4), dim3(256), 0, st, a, c);
  }
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

}  // namespace

void launch_window_dq(const BlockArgs &a, bool bf16, bool few, float *delta, float *logs, hipStream_t st) {
  const long long tiles = ceil_div((long long)a.block_m * a.group, few ? 16 : 128);
  const auto go = [&](auto type, auto dim) {
    typedef decltype(type) T;
    constexpr int DP = decltype(dim)::value;
    const bool sides = !few && few_workgroups(a);
    const auto kernel = few ? block_dq_narrow_kernel<T, DP, 4, true> : sides ? block_dq_kernel<T, DP, 4, 64, true, 2> : block_dq_kernel<T, DP, 4, 64, true>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((long long)a.batch * a.kv_heads * a.rows * tiles)), dim3(sides ? 512 : 256), 0, st, a, (int)tiles, delta, logs, nullptr);
  };
  const auto with = [&](auto type) {
    if (a.dim <= 64) go(type, std::integral_constant<int, 64>());
    else go(type, std::integral_constant<int, 128>());
  };
  if (bf16) with(Bf16());
  else with(F16());
}

}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_block_attention_backward_work(const lapis_hip_block_args *args, int64_t *bytes) {
  LAPIS_CHECK_INIT();  // the size goes by the number of compute units
  BlockArgs a;
  int rc = read_block("block_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "block_attention_backward: null result");
  Layout l;
  rc = layout_of(a, &l);
  *bytes = l.bytes;
  return rc;
}

extern "C" int lapis_hip_block_attention_backward(const lapis_hip_block_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_block("block_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0 || (a.heads == 0 && a.kv_heads == 0)) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(args->work && aligned16(args->work), "block_attention_backward: work that is null or not on a 16-byte boundary");
  char *work = static_cast<char *>(args->work);
  const bool bf16 = args->dtype == LAPIS_HIP_BF16;
  if (a.dim <= 64) return bf16 ? launch_backward<Bf16, 64>(a, work, as_stream(stream)) : launch_backward<F16, 64>(a, work, as_stream(stream));
  return bf16 ? launch_backward<Bf16, 128>(a, work, as_stream(stream)) : launch_backward<F16, 128>(a, work, as_stream(stream));
}
