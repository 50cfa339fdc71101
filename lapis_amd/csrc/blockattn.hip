// Attention over the blocks that a CSR structure lists, or over a window and the first keys, forward.
#include "blockattn.hpp"

namespace lapis {
namespace {

// Factor of scores in units of ln 2 (the sign goes to the queries): never 0, as masked scores are -infinity; NaN stays.
__device__ __forceinline__ float units_of_ln2(float scale) {
  const float c = fabsf(scale) * 1.4426950408889634f;
  return c < 1e-37f ? 1e-37f : c;
}

// Rows of a list are its queries times the heads of the group, heads first: row i is query i / group, head i % group.
//
// A workgroup takes 32 * NW rows of one list, a wavefront 32 of them.  Tiles of KT keys go through LDS (two buffers: the
// next tile is loaded straight into one while the other is computed).
// S^T = K Q^T has a query per lane, so maxima, sums and factors of the softmax are one register and need one exchange
// between the halves of the wavefront; P^T feeds O^T = V^T P^T from the registers it was computed in.  For that it is rounded to the operands' type, the one
// rounding before the result's own (the sums that divide it take it in 32 bits): products of 32-bit operands have a sixteenth of the rate.
// Operands from LDS are asked for some products ahead (a fence after each product keeps it so: left alone the compiler reads each pair of them and
// waits), and the two ways of taking values, with infinities and NaN apart and without, are no two sides of one branch (64 registers less).
// 32 768 queries and keys, 32 heads over 8, dim 128, bf16: 16 blocks of 128 a row 1120 to 1165 us, a window of 2048 and the first 16 keys 1116 to 1170
// (885 to 965 TFLOP/s where a large library product reaches 1203 to 1400).  Near the card's power: with operands that are zeros it
// is 20 % faster and that product 30 %; exponentials of half a tile under the products of the other half change nothing.
template <typename T, int DP, int NW, int KT, bool WINDOW, int SIDES = 1>
__global__ __launch_bounds__(64 * NW * SIDES, 2) void block_forward_kernel(BlockArgs a, int tiles_of_list, int flip) {
  typedef typename T::elem elem;
  constexpr int PIECES = DP / 8, PASSES = KT * PIECES / (NW * 64), ST = KT / 32, DT = DP / 32, CH = KT / 16;
  __shared__ __attribute__((aligned(16))) elem k_tile[SIDES][2][KT * DP], v_tile[SIDES][2][KT * DP];
  __shared__ int bad_tile[SIDES][2];
  const int tid = threadIdx.x % (64 * NW), side = SIDES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * NW)), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const unsigned block = xcd_contiguous_block(blockIdx.x, gridDim.x);
  const int list = block / tiles_of_list, part = block - list * tiles_of_list;
  const int bh = list / a.rows, r = list - bh * a.rows, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const int q0 = r * a.block_m, held = min(a.block_m, a.queries - q0), rows = held * a.group;
  if (part * 32 * NW >= rows) return;  // the last block of queries is cut
  int first = 0, count = 0;
  if (!WINDOW) entries_of(a, list, &first, &count);

  const int row0 = part * 32 * NW + wave * 32, row = row0 + (lane & 31);
  const bool live = row < rows;
  const int query = q0 + row / a.group, head = kh * a.group + row % a.group;
  const int limit = a.causal ? min(query + a.shift, a.keys - 1) : a.keys - 1;  // last key this row sees
  const int row_last = min(row0 + 31, rows - 1);
  const int low = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row0 / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int high = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row_last / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int low_of_all = a.causal ? min(q0 + part * 32 * NW / a.group + a.shift, a.keys - 1) : a.keys - 1;
  const int row_last_of_all = min(part * 32 * NW + 32 * NW, rows) - 1;
  const Sight<WINDOW> row_sees(a, limit);
  const int gone_any = high - a.window, gone_any_of_all = q0 + row_last_of_all / a.group + a.shift - a.window;

  vec8<T> qf[DP / 16];
  const elem *qp = (const elem *)a.q.data + b * a.q.stride[0] + query * a.q.stride[1] + head * a.q.stride[2];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * half;
    v4i x = {0, 0, 0, 0};
    if (live && d < a.dim) x = *(const v4i *)(qp + d);
    qf[s] = __builtin_bit_cast(vec8<T>, x ^ flip);
  }
  KeyTiles<T, DP, NW, KT, true, WINDOW> keys(a, b, kh, first, count, tid, k_tile[side][0], v_tile[side][0]);
  if (WINDOW) keys.span = span_of(a, q0, held);
  const int tiles = keys.tiles(), steps = SIDES == 1 ? tiles : (tiles + SIDES - 1) / SIDES;
  v4i now, next;  // first keys of each sixteen of this tile and the next

  v16f acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = v16f{};
  const float c = units_of_ln2(a.scale);
  float m = -INFINITY, l = 0.f;  // of this row; l of this half's keys

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
      for (int p = 0; p < PASSES; ++p) bad |= not_finite<T>(*(const vec8<T> *)(v_tile[side][buffer] + (p * NW * 64 + tid) * 8));
      if (__any(bad) && lane == 0) bad_tile[side][buffer] = t + 1;
      if (SIDES == 1) __syncthreads();
    }
    if (SIDES > 1) __syncthreads();  // of all, as one side's tile may be cut and not the other's
    if (lowest <= high) {
      const elem *kt = k_tile[side][buffer], *vt = v_tile[side][buffer];
      // keys by rows, read some products ahead; the chains of products of the tile's halves in turn
      constexpr int KN = ST * DP / 16, K_AHEAD = 4;
      v16f s[ST] = {};
      vec8<T> ka[KN];
      const auto read_keys = [&](int n) { ka[n] = *(const vec8<T> *)(kt + place_of<DP>(32 * (n % ST) + (lane & 31), 2 * (n / ST) + half)); };
#pragma unroll
      for (int n = 0; n < K_AHEAD; ++n) read_keys(n);
      const auto score = [&](int n) {
        if (n + K_AHEAD < KN) read_keys(n + K_AHEAD);
        s[n % ST] = mfma32(ka[n], qf[n / ST], s[n % ST]);
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int n = 0; n < KN * 3 / 4; ++n) score(n);
      if (DP <= 64 || a.dim > 96) {  // the last quarter of a row, if it is there (dim 96, 8192 queries, window 1024: 188 us with it, 178 without; dim 128 the same)
#pragma unroll
        for (int n = KN * 3 / 4; n < KN; ++n) score(n);
      }
      const bool cut = top + 15 > low || (WINDOW && lowest <= gone_any);
      int clean = 1;
      if (cut) {
        clean = bad_tile[side][buffer] != t + 1;
#pragma unroll
        for (int x = 0; x < ST; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = now[2 * x + (e >> 3)] + 8 * ((e >> 2) & 1) + 4 * half + (e & 3);
            s[x][e] = row_sees.sees(key) ? s[x][e] : -INFINITY;
          }
      }
      float best = s[0][0];
#pragma unroll
      for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) best = fmaxf(best, s[x][e]);
      best = halves_max(best) * c;
      // the maximum in use moves only when it is left behind by more than 2^8: P stays below that, exact in fp32
      if (__any(best > m + 8.f)) {
        const float to = fmaxf(m, best), keep = to == m ? 1.f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= keep;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] *= keep;
      }
      const float off = m == -INFINITY ? 0.f : m;
      // values by columns, read some products ahead, the first of them before the exponentials
      constexpr int N = 2 * ST * DT, AHEAD = 4;
      vec8<T> pf[2 * ST], va[N];
      constexpr int LAST = DP <= 64 ? 0 : N / DT, FIRST = N - LAST;  // products of the last 32 columns come last
      const auto key_of = [](int n) { return n < FIRST ? n / (FIRST * DT / N) : n - FIRST; };
      const auto column_of = [](int n) { return n < FIRST ? n % (FIRST * DT / N) : DT - 1; };
      const auto read = [&](int n) { va[n] = columns_in_order<T, DP, true>(vt, 16 * key_of(n), 32 * column_of(n), lane); };
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) read(n);
#pragma unroll
      for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e] = __builtin_fmaf(s[x][e], c, -off);
#pragma unroll
      for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e] = __builtin_amdgcn_exp2f(s[x][e]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          l += s[x][e];
          pf[2 * x + (e >> 3)][e & 7] = (elem)s[x][e];
        }
      if (clean) {  // either way, but not as two sides of one branch: the sums would be kept twice
        const auto product = [&](int n) {
          if (n + AHEAD < N) read(n + AHEAD);
          acc[column_of(n)] = mfma32(va[n], pf[key_of(n)], acc[column_of(n)]);
          __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int n = 0; n < FIRST; ++n) product(n);
        if (LAST && a.dim > 96) {
#pragma unroll
          for (int n = FIRST; n < N; ++n) product(n);
        }
      }
      asm volatile("" : "+v"(clean));
      if (__builtin_amdgcn_readfirstlane(clean) == 0) {
        // the finite values as always; an infinity or NaN only to the rows that see its key
#pragma unroll
        for (int y = 0; y < 2 * ST; ++y)
#pragma unroll
          for (int i = 0; i < DT; ++i)
            acc[i] = mfma32(finite_only<T>(columns_in_order<T, DP, true>(vt, 16 * y, 32 * i, lane)), pf[y], acc[i]);
#pragma unroll 1
        for (int x = 0; x < KT; ++x) {
          int key0 = now[0];
#pragma unroll
          for (int i = 1; i < CH; ++i) key0 = x >> 4 == i ? now[i] : key0;
          const int key = key0 + (x & 15);
          const bool sees = row_sees.sees(key);
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const vec4<T> v = *(const vec4<T> *)(vt + place_of<DP, true>(x, 4 * i + (e >> 2)) + 4 * half);
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                const float f = (float)v[n];
                if (sees && abs_bits(f) >= kInfBits) acc[i][e + n] += f;
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

  l = halves_sum(l);
  if constexpr (SIDES > 1) {  // (the last step has ended with a barrier)
    float *sums = (float *)k_tile + wave * (DT * 1024) + lane * 4;
    float *rows_of_wave = (float *)v_tile + wave * 128 + lane;
    if (side) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) *(v4f *)(sums + (4 * i + e / 4) * 256) = v4f{acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]};
      rows_of_wave[0] = m;
      rows_of_wave[64] = l;
    }
    __syncthreads();
    if (side) return;
    const float other = rows_of_wave[0], most = fmaxf(m, other), off = most == -INFINITY ? 0.f : most;
    const float mine = __builtin_amdgcn_exp2f(m - off), theirs = __builtin_amdgcn_exp2f(other - off);
    l = l * mine + rows_of_wave[64] * theirs;
    m = most;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] = acc[i][e] * mine + sums[(4 * i + e / 4) * 256 + e % 4] * theirs;
  }
  const float factor = l == 0.f ? 0.f : 1.f / l;
  if (!live) return;
  elem *op = (elem *)a.out.data + b * a.out.stride[0] + query * a.out.stride[1] + head * a.out.stride[2];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * i + 2 * e + 4 * half;
      vec4<T> x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (elem)(l == 0.f ? 0.f : acc[i][e + j] * factor);
      if (d < a.dim) *(vec4<T> *)(op + d) = x;
    }
  if (a.lse && half == 0)
    a.lse[((long long)b * a.heads + head) * a.queries + query] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// Lists of few rows (queries of their own lists: a row block of one query has a row for each head of the group).  16 rows a
// wavefront, which reads its keys and values by itself: K from memory into the operand's registers (16x16x32, S^T = K Q^T, a
// row per lane), V through LDS, where it is read by columns, 32 keys at a time, the next ones loaded as soon as the
// registers are free.  SPLIT wavefronts share the keys of one list, by tiles in turn, and join through LDS.
// 4096 queries, 16 heads each over 16 blocks of 32 of their own, dim 64, f16: 82 us; 1.07 GB of keys and values out of L2 at 13 TB/s.
template <typename T, int DP, int SPLIT, bool WINDOW>
__global__ __launch_bounds__(256, DP <= 64 ? 4 : 2) void block_narrow_kernel(BlockArgs a, int tiles_of_list, int flip) {
  typedef typename T::elem elem;
  constexpr int KS = DP / 32, DT = DP / 16, PIECES = DP / 8, RP = 64 / PIECES, PASSES = 32 / RP;
  union Own {  // of a wavefront
    elem v[32 * DP];
    float out[16][DP + 4];
  };
  __shared__ __attribute__((aligned(16))) Own own[4];
  __shared__ float tops[4][16], totals[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quarter = lane >> 4;
  const int block = (int)(xcd_contiguous_block(blockIdx.x, gridDim.x) * (4 / SPLIT)) + wave / SPLIT, share = wave % SPLIT;
  const int list = block / tiles_of_list, part = block - list * tiles_of_list;
  const int lists = a.batch * a.kv_heads * a.rows;
  const bool any = list < lists;
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

  vec8<T> qf[KS];
  const elem *qp = (const elem *)a.q.data + b * a.q.stride[0] + query * a.q.stride[1] + head * a.q.stride[2];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 32 * s + 8 * quarter;
    v4i x = {0, 0, 0, 0};
    if (live && d < a.dim) x = *(const v4i *)(qp + d);
    qf[s] = __builtin_bit_cast(vec8<T>, x ^ flip);
  }
  const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + kh * a.k.stride[2];
  const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + kh * a.v.stride[2];
  const Sight<WINDOW> row_sees(a, limit);
  const int gone_any = high - a.window;  // last key before any row's window
  const int tiles = WINDOW ? (span.count + 1) / 2 : tiles_of<32>(a, count);
  const int piece = lane % PIECES, v_row = lane / PIECES, vd = piece * 8 < a.dim ? piece * 8 : 0;
  v4i kr[2][KS], vr[PASSES];
  const auto load = [&](const int (&key0)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int from = min(key0[i], a.keys - 1), room = a.keys - 1 - from;
      const elem *k = kp + from * a.k.stride[1] + min(col, room) * a.k.stride[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 32 * s + 8 * quarter;
        kr[i][s] = *(const v4i *)(k + (d < a.dim ? d : 0));
        if (a.dim < 32 * s + 32 && d >= a.dim) kr[i][s] = v4i{0, 0, 0, 0};
      }
#pragma unroll
      for (int p = i * PASSES / 2; p < (i + 1) * PASSES / 2; ++p)
        vr[p] = *(const v4i *)(vp + from * a.v.stride[1] + min((p * RP & 15) + v_row, room) * a.v.stride[1] + vd);
    }
  };
  const auto look_up = [&](int t) {
    if constexpr (WINDOW) return span.first_key(2 * t + (lane & 1));
    return tiles > 0 ? first_key(a, first, count, 32ll * t + 16 * (lane & 1)) : kAbsent;
  };

  v4f acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  const float c = units_of_ln2(a.scale);
  float m = -INFINITY, l = 0.f;
  elem *mine = own[wave].v;
  int now[2], next[2], ahead = look_up(share);
  next[0] = __builtin_amdgcn_readlane(ahead, 0), next[1] = __builtin_amdgcn_readlane(ahead, 1);
  if (share < tiles) load(next);
  ahead = look_up(share + SPLIT);
  for (int t = share; t < tiles; t += SPLIT) {
    now[0] = next[0], now[1] = next[1];
    v4f s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) s[i] = mfma16(__builtin_bit_cast(vec8<T>, kr[i][x]), qf[x], s[i]);
    }
    const bool cut = max(now[0], now[1]) + 15 > low || (WINDOW && min(now[0], now[1]) <= gone_any), skip = min(now[0], now[1]) > high;
    bool bad = false;
    if (cut) {  // 0 times an infinity or NaN must not count
#pragma unroll
      for (int p = 0; p < PASSES; ++p) bad |= not_finite<T>(__builtin_bit_cast(vec8<T>, vr[p]));
      bad = __any(bad);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int at = p * RP + v_row;
      *(v4i *)(mine + at * DP + ((piece ^ turn16<DP>(at)) * 8)) = vr[p];
    }
    next[0] = __builtin_amdgcn_readlane(ahead, 0), next[1] = __builtin_amdgcn_readlane(ahead, 1);
    if (t + SPLIT < tiles) load(next);
    ahead = look_up(t + 2 * SPLIT);
    if (skip) continue;
    if (cut) {
      asm volatile("");  // (one branch, not one for each element)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = row_sees.sees(now[i] + 4 * quarter + e) ? s[i][e] : -INFINITY;
    }
    wave_lds_sync();
    vec8<T> pf, va[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) {  // asked for before the exponentials
      const int x = 4 * quarter + (col >> 2), d = 16 * i + 4 * (col & 3);
      const elem *p = mine + x * DP + ((d >> 3) ^ turn16<DP>(x)) * 8 + (d & 7);  // row + 16 has the same order of pieces
      va[i] = join<T>(read_columns<T>(p), read_columns<T>(p + 16 * DP));
    }
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) best = fmaxf(best, s[i][e]);
    best = rows_max(best) * c;
    if (__any(best > m + 8.f)) {  // as in the kernel above
      const float to = fmaxf(m, best), keep = to == m ? 1.f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= keep;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] *= keep;
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], c, -off));
        l += p;
        pf[4 * i + e] = (elem)p;
      }
    if (bad) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < DT; ++i) va[i] = finite_only<T>(va[i]);
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = mfma16(va[i], pf, acc[i]);
    if (bad)  // an infinity or NaN only to the rows that see its key
#pragma unroll 1
      for (int x = 0; x < 32; ++x) {
        const int key = (x < 16 ? now[0] : now[1]) + (x & 15);
        const bool sees = row_sees.sees(key);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const int d = 16 * i + 4 * quarter;
          const vec4<T> v = *(const vec4<T> *)(mine + x * DP + ((d >> 3) ^ turn16<DP>(x)) * 8 + (d & 7));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sees && abs_bits((float)v[e]) >= kInfBits) acc[i][e] += (float)v[e];
        }
      }
    wave_lds_sync();
  }
  l = rows_sum(l);
  if (quarter == 0) tops[wave][col] = m, totals[wave][col] = l;
#pragma unroll
  for (int i = 0; i < DT; ++i) *(v4f *)(&own[wave].out[col][16 * i + 4 * quarter]) = acc[i];
  if (SPLIT == 1) wave_lds_sync();
  else __syncthreads();
  if (!any) return;
  // a piece of a row per lane, from all wavefronts that share the list
  constexpr int W0 = SPLIT == 1 ? 0 : 1;
  const int w0 = SPLIT == 1 ? wave : 0;
  for (int x = SPLIT == 1 ? lane : tid; x < 16 * PIECES; x += SPLIT * 64) {
    const int h = x / PIECES, d = (x % PIECES) * 8;
    if (row0 + h >= rows || d >= a.dim) continue;
    float most = tops[w0][h], sum = 0.f, o[8] = {};
#pragma unroll
    for (int w = W0; w < SPLIT; ++w) most = fmaxf(most, tops[w0 + w][h]);
#pragma unroll
    for (int w = 0; w < SPLIT; ++w) {
      const float by = tops[w0 + w][h] == most ? 1.f : __builtin_amdgcn_exp2f(tops[w0 + w][h] - most);
      sum += by * totals[w0 + w][h];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += by * own[w0 + w].out[h][d + e];
    }
    const float by = 1.f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = sum == 0.f ? 0.f : o[e] * by;
    const int i = q0 + (row0 + h) / a.group, to = kh * a.group + (row0 + h) % a.group;
    *(vec8<T> *)((elem *)a.out.data + b * a.out.stride[0] + i * a.out.stride[1] + to * a.out.stride[2] + d) = narrow<T>(o);
    if (a.lse && d == 0)
      a.lse[((long long)b * a.heads + to) * a.queries + i] = sum == 0.f ? -INFINITY : (most + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
  }
}

int read_view(const char *what, const lapis_hip_rows &r, View *v) {
  LAPIS_REQUIRE(r.data && aligned16(r.data) && strides_of_8(r.stride, 3),
                "%s: an operand that is null, not on a 16-byte boundary or with strides that are no multiples of 8", what);
  v->data = static_cast<char *>(r.data);
  for (int i = 0; i < 3; ++i) v->stride[i] = r.stride[i];
  return LAPIS_HIP_OK;
}

template <typename T, int DP, int NW, int KT, bool WINDOW, int SIDES = 1>
int launch_wide(const BlockArgs &a, hipStream_t st) {
  const long long lists = (long long)a.batch * a.kv_heads * a.rows, tiles = ceil_div((long long)std::min(a.block_m, a.queries) * a.group, 32 * NW);
  LAPIS_REQUIRE(lists * tiles * 64 * NW * SIDES < (INT64_C(1) << 32), WINDOW ? "window_attention: %lld rows" : "block_attention: %lld rows of the structure", lists);
  hipLaunchKernelGGL((block_forward_kernel<T, DP, NW, KT, WINDOW, SIDES>), dim3((unsigned)(lists * tiles)), dim3(64 * NW * SIDES), 0, st, a, (int)tiles,
                     a.scale < 0.f ? (int)0x80008000u : 0);
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

template <typename T, int DP, int SPLIT, bool WINDOW>
int launch_narrow(const BlockArgs &a, hipStream_t st) {
  const long long lists = (long long)a.batch * a.kv_heads * a.rows, tiles = ceil_div((long long)a.block_m * a.group, 16);
  const long long blocks = ceil_div(lists * tiles * SPLIT, 4);
  LAPIS_REQUIRE(blocks * 256 < (INT64_C(1) << 32), WINDOW ? "window_attention: %lld rows" : "block_attention: %lld rows of the structure", lists);
  hipLaunchKernelGGL((block_narrow_kernel<T, DP, SPLIT, WINDOW>), dim3((unsigned)blocks), dim3(256), 0, st, a, (int)tiles, a.scale < 0.f ? (int)0x80008000u : 0);
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

template <typename T>
int launch_forward(const BlockArgs &a, hipStream_t st) {
  // Up to 32 rows a list the 128-row workgroup mostly waits for its own tiles (16 rows, 4096 queries, 4 lists of 512 keys each, dim
  // 64: 498 us against 169; 32 rows: 257 against 167; 48 rows: 37.5 against 41.7), and while there are fewer of them than half
  // the compute units, 16 rows of four wavefronts spread further (128 rows, 64 workgroups: 10.5 against 8.2).
  const int64_t rows = (int64_t)a.block_m * a.group, lists = (int64_t)a.batch * a.kv_heads * a.rows, waves = ceil_div(rows, 16) * lists;
  if (rows <= 32 || ceil_div(rows, 128) * lists < device_cu_count() / 2) {
    const bool many = waves >= 8 * device_cu_count();  // two wavefronts a SIMD without sharing lists
    if (a.dim <= 64) return many ? launch_narrow<T, 64, 1, false>(a, st) : launch_narrow<T, 64, 4, false>(a, st);
    return many ? launch_narrow<T, 128, 1, false>(a, st) : launch_narrow<T, 128, 4, false>(a, st);
  }
  return a.dim <= 64 ? launch_wide<T, 64, 4, 64, false>(a, st) : launch_wide<T, 128, 4, 64, false>(a, st);
}

template <typename T>
int launch_window(BlockArgs a, hipStream_t st) {
  cut_queries(&a, 128);
  // the same rule
  if ((int64_t)a.batch * a.kv_heads * a.rows * ceil_div(a.block_m * a.group, 128) < device_cu_count() / 2) {
    cut_queries(&a, 16);
    return a.dim <= 64 ? launch_narrow<T, 64, 4, true>(a, st) : launch_narrow<T, 128, 4, true>(a, st);
  }
  if (few_workgroups(a)) return a.dim <= 64 ? launch_wide<T, 64, 4, 64, true, 2>(a, st) : launch_wide<T, 128, 4, 64, true, 2>(a, st);
  return a.dim <= 64 ? launch_wide<T, 64, 4, 64, true>(a, st) : launch_wide<T, 128, 4, 64, true>(a, st);
}

}  // namespace

int read_block(const char *what, const lapis_hip_block_args *p, bool backward, BlockArgs *a) {
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  LAPIS_REQUIRE(p->batch >= 0 && p->queries >= 0 && p->keys >= 0 && p->heads >= 0 && p->kv_heads >= 0, "%s: a negative size", what);
  LAPIS_REQUIRE(p->batch <= 65535 && p->heads <= 65535 && p->queries <= (1 << 30) && p->keys <= (1 << 30), "%s: %lld x %lld queries, %lld keys, %lld heads",
                what, (long long)p->batch, (long long)p->queries, (long long)p->keys, (long long)p->heads);
  LAPIS_REQUIRE((p->kv_heads == 0 && p->heads == 0) || (p->kv_heads > 0 && p->heads % p->kv_heads == 0), "%s: %lld heads over %lld key-value heads", what,
                (long long)p->heads, (long long)p->kv_heads);
  LAPIS_REQUIRE(p->dim >= 8 && p->dim <= kMaxBlockDim && p->dim % 8 == 0, "%s: rows of %lld elements (a multiple of 8 up to %d)", what,
                (long long)p->dim, kMaxBlockDim);
  LAPIS_REQUIRE(p->block_m >= 1 && p->block_m <= (1 << 30), "%s: blocks of %lld queries", what, (long long)p->block_m);
  LAPIS_REQUIRE(p->block_n >= 16 && p->block_n <= 256 && (p->block_n & (p->block_n - 1)) == 0, "%s: blocks of %lld keys (16, 32, 64, 128 or 256)", what,
                (long long)p->block_n);
  LAPIS_REQUIRE(p->nnz >= 0 && p->nnz <= INT32_MAX, "%s: %lld entries", what, (long long)p->nnz);
  LAPIS_REQUIRE(is_16bit(p->dtype), "%s: operands of type %d", what, p->dtype);
  *a = {};
  a->batch = (int)p->batch;
  a->queries = (int)p->queries;
  a->keys = (int)p->keys;
  a->heads = (int)p->heads;
  a->kv_heads = (int)p->kv_heads;
  a->group = p->kv_heads ? (int)(p->heads / p->kv_heads) : 0;
  a->dim = (int)p->dim;
  a->block_m = (int)std::min(p->block_m, std::max(p->queries, INT64_C(1)));  // a longer block has no more queries
  a->block_n_log2 = __builtin_ctz((unsigned)p->block_n);
  a->rows = (int)ceil_div(p->queries, p->block_m);
  a->columns = (int)ceil_div(p->keys, p->block_n);
  if (p->heads == 0) a->rows = 0, a->group = 1;
  a->causal = p->causal != 0;
  a->shift = (int)(p->keys - p->queries);
  a->scale = p->scale;
  a->pos = p->pos;
  a->crd = p->crd;
  a->nnz = a->rows ? p->nnz : 0;
  a->lse = p->lse;
  LAPIS_REQUIRE(!backward || (double)p->batch * (double)p->heads * (double)p->queries < 2147483647.0, "%s: more queries times heads than 31 bits count", what);
  LAPIS_REQUIRE((double)p->batch * (double)p->kv_heads * (double)a->rows < 2147483647.0, "%s: more rows than 31 bits count", what);
  const bool some_queries = p->batch && p->queries && p->heads, some_keys = p->batch && p->keys && p->kv_heads;
  if (some_queries || (backward && some_keys && p->queries)) LAPIS_REQUIRE(p->pos && (p->crd || p->nnz == 0), "%s: null structure", what);
  LAPIS_REQUIRE(!backward || !some_queries || p->lse, "%s: null lse", what);
  int rc = LAPIS_HIP_OK;
  const auto take = [&](bool some, const lapis_hip_rows &r, View *v) {
    if (some && rc == LAPIS_HIP_OK) rc = read_view(what, r, v);
  };
  take(some_queries, p->q, &a->q);
  take(some_keys, p->k, &a->k);
  take(some_keys, p->v, &a->v);
  take(some_queries, p->out, &a->out);
  if (backward) {
    take(some_queries, p->dout, &a->dout);
    take(some_queries, p->dq, &a->dq);
    take(some_keys, p->dk, &a->dk);
    take(some_keys, p->dv, &a->dv);
  }
  return rc;
}

int read_window(const char *what, const lapis_hip_window_args *p, bool backward, BlockArgs *a) {
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  LAPIS_REQUIRE(p->window >= 1 && p->sink >= 0, "%s: a window of %lld and the first %lld keys", what, (long long)p->window, (long long)p->sink);
  static const int32_t none = 0;  // of lists, which are not looked at
  lapis_hip_block_args b = {};
  b.batch = p->batch, b.queries = p->queries, b.keys = p->keys, b.heads = p->heads, b.kv_heads = p->kv_heads, b.dim = p->dim;
  b.block_m = 1, b.block_n = 64;
  b.causal = 1, b.dtype = p->dtype, b.scale = p->scale;
  b.pos = b.crd = &none;
  b.q = p->q, b.k = p->k, b.v = p->v, b.out = p->out, b.lse = p->lse;
  b.dout = p->dout, b.dq = p->dq, b.dk = p->dk, b.dv = p->dv;
  const int rc = read_block(what, &b, backward, a);
  a->pos = a->crd = nullptr;
  if (p->heads == 0) a->queries = 0;  // queries without a head are no rows: nothing of q is there to be read
  // positions, and what is taken from them, stay within 32 bits
  a->window = (int)std::min<int64_t>(p->window, 1 << 30);
  a->sink = (int)std::min<int64_t>(p->sink, 1 << 30);
  return rc;
}

}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_block_attention(const lapis_hip_block_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_block("block_attention", args, false, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0 || a.queries == 0 || a.heads == 0) return LAPIS_HIP_OK;
  return args->dtype == LAPIS_HIP_BF16 ? launch_forward<Bf16>(a, as_stream(stream)) : launch_forward<F16>(a, as_stream(stream));
}

extern "C" int lapis_hip_window_attention(const lapis_hip_window_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_window("window_attention", args, false, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0 || a.queries == 0 || a.heads == 0) return LAPIS_HIP_OK;
  return args->dtype == LAPIS_HIP_BF16 ? launch_window<Bf16>(a, as_stream(stream)) : launch_window<F16>(a, as_stream(stream));
}
