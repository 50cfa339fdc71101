// Attention over the blocks that a CSR structure lists, backward.
//
// P and dS are computed twice, once beside dQ (rows of the structure, as in the forward pass) and once beside dK and dV
// (its columns): nothing is added by atomics, so the same inputs give the same bits.  The columns' lists of rows are made
// here (counted, summed, filled: three small kernels), since a selection is another one in every training step.
#include "blockattn.hpp"

namespace lapis {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---- dQ --------------------------------------------------------------------------------------------------------

// As the forward kernel: 32 rows a wavefront, a query per lane.  dS^T = P^T * (scale V dO^T - scale delta) feeds dQ^T = K^T dS^T
// from its registers.  rowsum(dO * O) is computed here and left, times `scale`, for the other kernel.
template <typename T, int DP, int NW, int KT>
__global__ __launch_bounds__(64 * NW, 2) void block_dq_kernel(BlockArgs a, int tiles_of_list, float *__restrict__ delta) {
  typedef typename T::elem elem;
  constexpr int PIECES = DP / 8, PASSES = KT * PIECES / (NW * 64), ST = KT / 32, DT = DP / 32, CH = KT / 16;
  __shared__ __attribute__((aligned(16))) elem k_tile[2][KT * DP], v_tile[2][KT * DP];
  __shared__ int bad_tile[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const unsigned block = xcd_contiguous_block(blockIdx.x, gridDim.x);
  const int list = block / tiles_of_list, part = block - list * tiles_of_list;
  const int bh = list / a.rows, r = list - bh * a.rows, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const int q0 = r * a.block_m, held = min(a.block_m, a.queries - q0), rows = held * a.group;
  if (part * 32 * NW >= rows) return;
  int first, count;
  entries_of(a, list, &first, &count);

  const int row0 = part * 32 * NW + wave * 32, row = row0 + (lane & 31);
  const bool live = row < rows;
  const int query = q0 + row / a.group, head = kh * a.group + row % a.group;
  const int limit = a.causal ? min(query + a.shift, a.keys - 1) : a.keys - 1;
  const int row_last = min(row0 + 31, rows - 1);
  const int low = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row0 / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int high = __builtin_amdgcn_readfirstlane(a.causal ? min(q0 + row_last / a.group + a.shift, a.keys - 1) : a.keys - 1);
  const int low_of_all = a.causal ? min(q0 + part * 32 * NW / a.group + a.shift, a.keys - 1) : a.keys - 1;

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
    if (half == 0) delta[at] = del;
  }
  const KeyTiles<T, DP, NW, KT, false> keys(a, b, kh, first, count, tid, k_tile[0], v_tile[0]);
  const int tiles = keys.tiles();
  int next[CH], now[CH];
  v16f acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = v16f{};
  const float c = a.scale * kLog2e;

  if (tid < 2) bad_tile[tid] = 0;
  if (a.dim < DP) {  // what no row fills stays zero
    for (int i = tid; i < 2 * KT * PIECES; i += 64 * NW) ((v4i *)k_tile)[i] = ((v4i *)v_tile)[i] = v4i{0, 0, 0, 0};
    __syncthreads();
  }
  if (tiles > 0) keys.load(0, next);
  lds_loads_done();
  __syncthreads();
  for (int t = 0; t < tiles; ++t) {
#pragma unroll
    for (int i = 0; i < CH; ++i) now[i] = next[i];
    if (t + 1 < tiles) keys.load(t + 1, next);
    int lowest = now[0], top = now[0];
#pragma unroll
    for (int i = 1; i < CH; ++i) lowest = min(lowest, now[i]), top = max(top, now[i]);
    if (top + 15 > low_of_all) {  // somebody's mask cuts this tile: 0 times an infinity or NaN must not count
      bool bad = false;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) bad |= not_finite<T>(*(const vec8<T> *)(k_tile[t & 1] + (p * NW * 64 + tid) * 8));
      if (__any(bad) && lane == 0) bad_tile[t & 1] = t + 1;
      __syncthreads();
    }
    if (lowest <= high) {
      const elem *kt = k_tile[t & 1], *vt = v_tile[t & 1];
      const bool cut = top + 15 > low;
      const bool bad = cut && bad_tile[t & 1] == t + 1;
#pragma unroll
      for (int x = 0; x < ST; ++x) {
        v16f s = {}, g = {};
#pragma unroll
        for (int y = 0; y < DP / 16; ++y) s = mfma32(*(const vec8<T> *)(kt + place_of<DP>(32 * x + (lane & 31), 2 * y + half)), qf[y], s);
#pragma unroll
        for (int y = 0; y < DP / 16; ++y) g = mfma32(*(const vec8<T> *)(vt + place_of<DP>(32 * x + (lane & 31), 2 * y + half)), gf[y], g);
        vec8<T> df[2];
        // dS is rounded to the operands' type for the product, with `scale` in it: smaller by its factor in float16's range
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -off));
          float ds = p * __builtin_fmaf(g[e], a.scale, -del);
          if (cut) {
            const int key = now[2 * x + (e >> 3)] + 8 * ((e >> 2) & 1) + 4 * half + (e & 3);
            ds = key > limit ? 0.f : ds;
          }
          df[e >> 3][e & 7] = (elem)ds;
        }
        // a row that sees a key with an infinity or NaN has NaN in its score; the others take the key as zeros
        if (bad) {
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < DT; ++i)
              acc[i] = mfma32(finite_only<T>(columns_in_order<T, DP>(kt, 32 * x + 16 * y, 32 * i, lane)), df[y], acc[i]);
        } else {
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] = mfma32(columns_in_order<T, DP>(kt, 32 * x + 16 * y, 32 * i, lane), df[y], acc[i]);
        }
      }
    }
    lds_loads_done();
    __syncthreads();
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

// ---- the columns' lists ----------------------------------------------------------------------------------------

// Which rows list a column, in ascending order (a row that lists it twice, twice).  Rows are cut into at most 32 chunks;
// counts[column][chunk], summed over a (batch entry, head)'s columns and chunks, gives each chunk its places.
struct Columns {
  int *odd;           // not 0: positions overlap or leave [0, nnz]; the lists are not used then
  int *counts;        // lists x columns x chunks
  int *start, *end;   // of each column's rows
  int *unit;          // column of each unit of work, -1 = nothing to do
  int *rows;          // nnz
  float *partial;     // of columns of several units: dk and dv of each
  int chunks, chunk_rows, per_unit, units, lists, sub;
};

constexpr int kColumnsInLds = 8192;

template <bool FILL>
__global__ __launch_bounds__(64) void columns_kernel(BlockArgs a, Columns t) {
  __shared__ int place[kColumnsInLds];
  const int lane = threadIdx.x, chunk = blockIdx.x, bh = blockIdx.z;
  const int c0 = blockIdx.y * kColumnsInLds, cs = min(kColumnsInLds, a.columns - c0);
  for (int c = lane; c < cs; c += 64) place[c] = FILL ? t.counts[((long long)bh * a.columns + c0 + c) * t.chunks + chunk] : 0;
  __syncthreads();
  const int r_end = min(a.rows, (chunk + 1) * t.chunk_rows);
  bool odd = false;
  for (int r = chunk * t.chunk_rows; r < r_end; ++r) {
    const long long row = (long long)bh * a.rows + r;
    int first, count;
    entries_of(a, row, &first, &count);
    odd |= a.pos[row] != first || (long long)a.pos[row + 1] != (long long)first + count;
    // one wavefront, row after row: the places of a column ascend with its rows
    for (int e = lane; e < count; e += 64) {
      const int c = a.crd[first + e];
      if ((unsigned)c < (unsigned)a.columns && c >= c0 && c < c0 + cs) {
        const int at = atomicAdd(&place[c - c0], 1);
        if (FILL && at < a.nnz) t.rows[at] = r;
      }
    }
    __syncthreads();
  }
  if (FILL) return;
  if (odd && lane == 0) atomicOr(t.odd, 1);
  for (int c = lane; c < cs; c += 64) t.counts[((long long)bh * a.columns + c0 + c) * t.chunks + chunk] = place[c];
}

__global__ void clear_kernel(int *p) { *p = 0; }

// Where a list's entries start (positions are in order here).
__device__ __forceinline__ int list_start(const BlockArgs &a, long long bh) {
  return a.rows ? (int)min(max((long long)a.pos[bh * a.rows], 0ll), a.nnz) : 0;
}

// One workgroup per (batch entry, key-value head): counts become places, columns get their ranges and their units of work.
__global__ __launch_bounds__(1024) void columns_scan_kernel(BlockArgs a, Columns t) {
  __shared__ int wave_sum[16], total;
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
    const int cc = bh * a.columns + c, start = t.start[cc], rows = t.end[cc] - start;
    const int needed = max(1, (rows + t.per_unit - 1) / t.per_unit);
    // the places start / per_unit + column leave each column at least as many units as it needs
    const long long to = (long long)start / t.per_unit + cc;
    const long long stop = c + 1 < a.columns  ? (long long)t.end[cc] / t.per_unit + cc + 1
                           : bh + 1 < t.lists ? (long long)list_start(a, bh + 1ll) / t.per_unit + cc + 1
                                              : t.units;
    for (long long u = to; u < stop && u < t.units; ++u) t.unit[u] = u < to + needed ? cc : -1;
  }
}

// ---- dK and dV -------------------------------------------------------------------------------------------------

// A workgroup takes 32 * KG keys of a column and some of the rows that list it, their queries times heads packed into tiles of
// 32: KG wavefronts share a tile, 4 / KG such groups take turns and add up at the end.  With a key per lane P and dS (queries x
// keys) feed dV^T = dO^T P and dK^T = Q^T dS from their registers; K and V of a wavefront's keys stay in registers.
// A tile's rows (where they lie, log-sums, deltas, last keys) are looked up while earlier ones are computed: place in the
// list two tiles ahead, sums one and a half, so that no wait is left but the one at the end of a tile.
template <typename T, int DP, int KG>
__global__ __launch_bounds__(256, 1) void block_dkv_kernel(BlockArgs a, Columns cols, const float *__restrict__ delta) {
  typedef typename T::elem elem;
  constexpr int QG = 4 / KG, PIECES = DP / 8, RP = KG * 64 / PIECES, PASSES = 32 / RP, DT = DP / 32;
  struct Info {
    long long q[32], g[32];
    float off[32], del[32];
    int last[32];
  };
  __shared__ __attribute__((aligned(16))) elem tiles[QG][2][2][32 * DP];
  __shared__ __attribute__((aligned(16))) Info infos[QG][3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int kg = wave % KG, qg = wave / KG, gt = tid - qg * KG * 64;
  const unsigned block = xcd_contiguous_block(blockIdx.x, gridDim.x);
  const int u = block / cols.sub, sub = block - u * cols.sub;
  const bool odd = *cols.odd != 0;
  int cc, from = 0, n, start = 0;
  bool several = false;
  if (odd) {  // every row is looked through for the column
    if (u >= cols.lists * a.columns) return;
    cc = u;
    n = a.rows;
  } else {
    cc = cols.unit[u];
    if (cc < 0) return;
    start = cols.start[cc];
    const int rows = cols.end[cc] - start;
    several = rows > cols.per_unit;
    from = (u - (start / cols.per_unit + cc)) * cols.per_unit;
    n = min(rows - from, cols.per_unit);
  }
  const int bh = cc / a.columns, column = cc - bh * a.columns, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const int in_block = sub * 32 * KG + kg * 32;
  const int key_low = (column << a.block_n_log2) + in_block, key = key_low + (lane & 31);
  const bool live = in_block + (lane & 31) < (1 << a.block_n_log2) && key < a.keys;

  vec8<T> kf[DP / 16], vf[DP / 16];
  const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + key * a.k.stride[1] + kh * a.k.stride[2];
  const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + key * a.v.stride[1] + kh * a.v.stride[2];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * half;
    kf[s] = vf[s] = vec8<T>{};
    if (live && d < a.dim) kf[s] = *(const vec8<T> *)(kp + d), vf[s] = *(const vec8<T> *)(vp + d);
  }

  // this lane's row of the tiles of its group: entry, query of the block and head of the group, moved on by 32 QG each tile
  const int steps_h = 32 * QG % a.group, steps_q = 32 * QG / a.group % a.block_m, steps_e = 32 * QG / a.group / a.block_m;
  const int slot0 = qg * 32 + (lane & 31);
  int entry = slot0 / a.group / a.block_m, in = slot0 / a.group % a.block_m, hd = slot0 % a.group;
  const auto on = [&] {
    hd += steps_h;
    in += steps_q;
    entry += steps_e;
    if (hd >= a.group) hd -= a.group, ++in;
    if (in >= a.block_m) in -= a.block_m, ++entry;
  };
  const long long all = (long long)n * a.block_m * a.group;
  const int tiles_n = (int)((all + 32 * QG - 1) / (32 * QG));

  int row_next = 0;  // list row of the tile after the one whose sums are on their way
  struct Row {
    int query, head;
    bool there;
    float weight;
  } now_row = {0, 0, false, 1.f};
  float lse_next = 0.f, del_next = 0.f;
  const auto fetch_row = [&] { row_next = odd || entry >= n ? entry : cols.rows[start + from + entry]; };
  const auto fetch_sums = [&] {  // of the row that fetch_row found; then on to the next tile's
    now_row.there = entry < n;
    now_row.query = row_next * a.block_m + in;
    now_row.there = now_row.there && now_row.query < a.queries;
    if (!now_row.there) now_row.query = 0;
    now_row.head = kh * a.group + hd;
    now_row.weight = 0.f;
    if (odd && now_row.there) {
      int first, count, times = 0;
      entries_of(a, (long long)bh * a.rows + row_next, &first, &count);
      for (int e = 0; e < count; ++e) times += a.crd[first + e] == column;
      now_row.weight = __builtin_amdgcn_logf((float)times);  // a row that does not list the column: -infinity, weight 0
    }
    const long long at = ((long long)b * a.heads + now_row.head) * a.queries + now_row.query;
    lse_next = a.lse[at];
    del_next = delta[at];
    on();
  };
  const auto put_info = [&](int t) {
    Info &i = infos[qg][t % 3];
    if (kg != 0 || lane >= 32) return;
    i.q[lane] = b * a.q.stride[0] + now_row.query * a.q.stride[1] + now_row.head * a.q.stride[2];
    i.g[lane] = b * a.dout.stride[0] + now_row.query * a.dout.stride[1] + now_row.head * a.dout.stride[2];
    i.off[lane] = !now_row.there || lse_next == -INFINITY ? INFINITY : lse_next * kLog2e - now_row.weight;
    i.del[lane] = del_next;
    i.last[lane] = !now_row.there ? -1 : a.causal ? min(now_row.query + a.shift, a.keys - 1) : a.keys - 1;
  };
  const int place = gt % PIECES, my_row = gt / PIECES;
  const auto load = [&](int t) {
    const Info &i = infos[qg][t % 3];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int at = p * RP + my_row, d = (place ^ turn<DP>(at)) * 8;
      const unsigned to = __builtin_amdgcn_readfirstlane((p * KG + kg) * 1024);
      if (d < a.dim) {
        load_to_lds((const elem *)a.q.data + i.q[at] + d, lds_address(tiles[qg][t & 1][0]) + to);
        load_to_lds((const elem *)a.dout.data + i.g[at] + d, lds_address(tiles[qg][t & 1][1]) + to);
      }
    }
  };

  v16f dk[DT], dv[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) dk[i] = dv[i] = v16f{};
  const float c = a.scale * kLog2e;
  if (a.dim < DP)
    for (int i = tid; i < QG * 4 * 32 * PIECES; i += 256) ((v4i *)tiles)[i] = v4i{0, 0, 0, 0};
  if (tiles_n > 0) {
    // tiles 0 and 1 looked up, tile 0 loaded, the sums of tile 2 and the row of tile 3 under way
    fetch_row();
    fetch_sums();
    put_info(0);
    fetch_row();
    fetch_sums();
    put_info(1);
    fetch_row();
    fetch_sums();
    fetch_row();
    __syncthreads();
    load(0);
  }
  lds_loads_done();
  __syncthreads();
  for (int t = 0; t < tiles_n; ++t) {
    put_info(t + 2);
    fetch_sums();
    fetch_row();
    if (t + 1 < tiles_n) load(t + 1);
    const Info &info = infos[qg][t % 3];
    const elem *qt = tiles[qg][t & 1][0], *gt_ = tiles[qg][t & 1][1];
    const int last = info.last[lane & 31];
    if (__any(last >= key_low)) {
      const bool cut = __any(last < key_low + 31);
      v16f s = {}, g = {};
#pragma unroll
      for (int y = 0; y < DP / 16; ++y) s = mfma32(*(const vec8<T> *)(qt + place_of<DP>(lane & 31, 2 * y + half)), kf[y], s);
#pragma unroll
      for (int y = 0; y < DP / 16; ++y) g = mfma32(*(const vec8<T> *)(gt_ + place_of<DP>(lane & 31, 2 * y + half)), vf[y], g);
      vec8<T> pf[2], df[2];
      bool bad = false;
      if (cut) {  // 0 times an infinity or NaN must not count
        for (int i = 0; i < PIECES / 2; ++i)
          bad |= not_finite<T>(*(const vec8<T> *)(qt + (i * 64 + lane) * 8)) || not_finite<T>(*(const vec8<T> *)(gt_ + (i * 64 + lane) * 8));
        bad = __any(bad);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4f off = *(const v4f *)(info.off + 8 * j + 4 * half), del = *(const v4f *)(info.del + 8 * j + 4 * half);
        const v4i lim = *(const v4i *)(info.last + 8 * j + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * j + e], c, -off[e]));
          float ds = p * __builtin_fmaf(g[4 * j + e], a.scale, -del[e]);
          if (bad && abs_bits(g[4 * j + e]) >= kInfBits) p = __builtin_nanf("");  // its row of dO is taken as zeros below
          if (cut && key > lim[e]) p = ds = 0.f;
          pf[j >> 1][(4 * j + e) & 7] = (elem)p;
          df[j >> 1][(4 * j + e) & 7] = (elem)ds;
        }
      }
      if (bad) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            dv[i] = mfma32(finite_only<T>(columns_in_order<T, DP>(gt_, 16 * y, 32 * i, lane)), pf[y], dv[i]);
            dk[i] = mfma32(finite_only<T>(columns_in_order<T, DP>(qt, 16 * y, 32 * i, lane)), df[y], dk[i]);
          }
      } else {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
          for (int i = 0; i < DT; ++i) dv[i] = mfma32(columns_in_order<T, DP>(gt_, 16 * y, 32 * i, lane), pf[y], dv[i]);
#pragma unroll
          for (int i = 0; i < DT; ++i) dk[i] = mfma32(columns_in_order<T, DP>(qt, 16 * y, 32 * i, lane), df[y], dk[i]);
        }
      }
    }
    lds_loads_done();
    __syncthreads();
  }

  // the groups' sums, in their order, with the tiles' memory between them
  if (QG > 1) {
    float *sums = (float *)tiles;  // (group - 1, key group): 2 DT 16 values of 64 lanes
    constexpr int EACH = 2 * DT * 16 * 64;
    static_assert((QG - 1) * KG * EACH / 2 * 4 <= (int)sizeof(tiles), "the groups' sums fit");
#pragma unroll
    for (int part = 0; part < 2; ++part) {  // dk, then dv
      if (part) __syncthreads();
      if (qg > 0) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) sums[((qg - 1) * KG + kg) * (EACH / 2) + (i * 16 + e) * 64 + lane] = part ? dv[i][e] : dk[i][e];
      }
      __syncthreads();
      if (qg == 0)
        for (int x = 0; x < QG - 1; ++x)
#pragma unroll
          for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float f = sums[(x * KG + kg) * (EACH / 2) + (i * 16 + e) * 64 + lane];
              if (part) dv[i][e] += f;
              else dk[i][e] += f;
            }
    }
  }
  if (qg > 0 || !live) return;
  if (several) {
    const long long slot = 2ll * (start / cols.per_unit) + from / cols.per_unit;
    float *to = cols.partial + (slot * 2 << a.block_n_log2) * DP + (long long)(in_block + (lane & 31)) * DP;
    float *to_v = to + ((long long)DP << a.block_n_log2);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * i + 2 * e + 4 * half;
        *(v4f *)(to + d) = v4f{dk[i][e], dk[i][e + 1], dk[i][e + 2], dk[i][e + 3]};
        *(v4f *)(to_v + d) = v4f{dv[i][e], dv[i][e + 1], dv[i][e + 2], dv[i][e + 3]};
      }
    return;
  }
  elem *kd = (elem *)a.dk.data + b * a.dk.stride[0] + key * a.dk.stride[1] + kh * a.dk.stride[2];
  elem *vd = (elem *)a.dv.data + b * a.dv.stride[0] + key * a.dv.stride[1] + kh * a.dv.stride[2];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * i + 2 * e + 4 * half;
      if (d >= a.dim) continue;
      vec4<T> x, y;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (elem)dk[i][e + j], y[j] = (elem)dv[i][e + j];
      *(vec4<T> *)(kd + d) = x;
      *(vec4<T> *)(vd + d) = y;
    }
}

// Columns of several units: their sums, in the order of the units.
template <typename T, int DP>
__global__ __launch_bounds__(256) void join_units_kernel(BlockArgs a, Columns cols) {
  typedef typename T::elem elem;
  const int cc = blockIdx.x;
  if (*cols.odd) return;
  const int start = cols.start[cc], rows = cols.end[cc] - start;
  if (rows <= cols.per_unit) return;
  const int units = (rows + cols.per_unit - 1) / cols.per_unit;
  const int bh = cc / a.columns, column = cc - bh * a.columns, b = bh / a.kv_heads, kh = bh - b * a.kv_heads;
  const long long each = (long long)DP << a.block_n_log2;
  const float *from = cols.partial + 2ll * (start / cols.per_unit) * 2 * each;
  for (long long x = threadIdx.x * 4; x < 2 * each; x += 1024) {
    const bool is_v = x >= each;
    const int at = (int)(is_v ? x - each : x), d = at % DP, key = (column << a.block_n_log2) + at / DP;
    if (key >= a.keys || d >= a.dim) continue;
    v4f sum = {0.f, 0.f, 0.f, 0.f};
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
  int64_t delta, odd, counts, start, end, unit, rows, partial, bytes;
  Columns columns;
};

Layout layout_of(const BlockArgs &a) {
  Layout l = {};
  Columns &c = l.columns;
  c.lists = a.batch * a.kv_heads;
  c.chunk_rows = (int)max((int64_t)64, ceil_div(a.rows, 32));
  c.chunks = (int)max((int64_t)1, ceil_div(a.rows, c.chunk_rows));
  // 4096 queries times heads a unit: a sixteenth of what a compute unit does in a large pass, so long columns do not stand alone
  const int64_t rows_of_entry = (int64_t)min(a.block_m, max(a.queries, 1)) * max(a.group, 1);
  c.per_unit = (int)max((int64_t)1, 4096 / rows_of_entry);
  c.units = (int)(a.nnz / c.per_unit + (int64_t)c.lists * a.columns);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.delta = take(4ll * a.batch * a.heads * a.queries);
  l.odd = take(4);
  l.counts = take(4ll * c.lists * a.columns * c.chunks);
  l.start = take(4ll * c.lists * a.columns);
  l.end = take(4ll * c.lists * a.columns);
  l.unit = take(4ll * c.units);
  l.rows = take(4 * a.nnz);
  const int dp = a.dim <= 64 ? 64 : 128;
  l.partial = take(2 * (a.nnz / c.per_unit) * 2 * ((int64_t)dp << a.block_n_log2) * 4);
  l.bytes = at;
  return l;
}

template <typename T, int DP, int KG>
void launch_dkv(const BlockArgs &a, const Columns &c, const float *delta, hipStream_t st) {
  Columns cols = c;
  cols.sub = (int)ceil_div(1 << a.block_n_log2, 32 * KG);
  hipLaunchKernelGGL((block_dkv_kernel<T, DP, KG>), dim3((unsigned)c.units * (unsigned)cols.sub), dim3(256), 0, st, a, cols, delta);
}

template <typename T, int DP>
int launch_backward(const BlockArgs &a, char *work, hipStream_t st) {
  Layout l = layout_of(a);
  Columns &c = l.columns;
  float *delta = reinterpret_cast<float *>(work + l.delta);
  c.odd = reinterpret_cast<int *>(work + l.odd);
  c.counts = reinterpret_cast<int *>(work + l.counts);
  c.start = reinterpret_cast<int *>(work + l.start);
  c.end = reinterpret_cast<int *>(work + l.end);
  c.unit = reinterpret_cast<int *>(work + l.unit);
  c.rows = reinterpret_cast<int *>(work + l.rows);
  c.partial = reinterpret_cast<float *>(work + l.partial);
  if (a.queries && a.heads) {
    const long long lists = (long long)c.lists * a.rows, tiles = ceil_div((long long)min(a.block_m, a.queries) * a.group, 128);
    LAPIS_REQUIRE(lists * tiles * 256 < (INT64_C(1) << 32), "block_attention_backward: %lld rows of the structure", lists);
    hipLaunchKernelGGL((block_dq_kernel<T, DP, 4, 64>), dim3((unsigned)(lists * tiles)), dim3(256), 0, st, a, (int)tiles, delta);
  }
  if (c.lists && a.columns) {
    hipLaunchKernelGGL(clear_kernel, dim3(1), dim3(1), 0, st, c.odd);
    const dim3 grid((unsigned)c.chunks, (unsigned)ceil_div(a.columns, kColumnsInLds), (unsigned)c.lists);
    LAPIS_REQUIRE(c.lists <= 65535 && (int64_t)c.units * 8 * 256 < (INT64_C(1) << 32), "block_attention_backward: %d lists, %d units", c.lists, c.units);
    hipLaunchKernelGGL(columns_kernel<false>, grid, dim3(64), 0, st, a, c);
    hipLaunchKernelGGL(columns_scan_kernel, dim3((unsigned)c.lists), dim3(1024), 0, st, a, c);
    hipLaunchKernelGGL(columns_kernel<true>, grid, dim3(64), 0, st, a, c);
    if (a.block_n_log2 <= 5) launch_dkv<T, DP, 1>(a, c, delta, st);
    else launch_dkv<T, DP, 2>(a, c, delta, st);
    hipLaunchKernelGGL((join_units_kernel<T, DP>), dim3((unsigned)(c.lists * a.columns)), dim3(256), 0, st, a, c);
  }
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_block_attention_backward_work(const lapis_hip_block_args *args, int64_t *bytes) {
  BlockArgs a;
  const int rc = read_block("block_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "block_attention_backward: null result");
  *bytes = layout_of(a).bytes;
  return LAPIS_HIP_OK;
}

extern "C" int lapis_hip_block_attention_backward(const lapis_hip_block_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_block("block_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0 || (a.heads == 0 && a.kv_heads == 0)) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(args->work, "block_attention_backward: null work");
  char *work = static_cast<char *>(args->work);
  const bool bf16 = args->dtype == LAPIS_HIP_BF16;
  if (a.dim <= 64) return bf16 ? launch_backward<Bf16, 64>(a, work, as_stream(stream)) : launch_backward<F16, 64>(a, work, as_stream(stream));
  return bf16 ? launch_backward<Bf16, 128>(a, work, as_stream(stream)) : launch_backward<F16, 128>(a, work, as_stream(stream));
}
