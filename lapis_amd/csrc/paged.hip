// Attention of one new token of each sequence over the pages of a cache that a CSR row lists, or over the window and the first tokens
// of a table of pages.
#include "kvcache.hpp"
#include "mfma.hpp"

namespace lapis {
namespace {

// What lists and windows need each for themselves lies in one place: arguments of four lines of 64 bytes, the grid's size behind them among it.  With a fifth
// line, which every workgroup waits for before it knows its unit, a call takes 0.1 to 0.5 us more (5 sequences of 628 tokens 10.1 us and 9.7, one of 34 4.5 and 4.3).
struct PagedArgs {
  const char *q;
  char *out;
  long long q_stride[2], out_stride[2];
  const char *k, *v;
  const void *k_scale, *v_scale;
  long long stride[3], scale_stride[3];
  long long pages;
  int seqs, heads, kv_heads, group, dim, page_log2;
  union {
    struct {
      const int *pos, *crd, *tokens;
      long long nnz;
      int rows;
      bool each;  // a list per key-value head
    } lists;
    struct {
      const int *table, *lengths;
      long long table_width;
      int window, sink, units_each;  // units of a sequence
    } windows;
  };
  bool windowed;
  float scale;
  float *lse;
  int chunk, units, head_tiles;  // pages (of windows: tokens) a unit, units of all lists, tiles of 16 heads
  float *partial, *sums;         // of each unit: 16 x DP, and 16 maxima and sums
};
static_assert(sizeof(PagedArgs) + sizeof(int) <= 256, "arguments and the number of workgroups in four lines");

// Pages that a row lists and tokens that count in them, whatever pos and tokens hold.
__device__ __forceinline__ void list_of(const PagedArgs &a, long long row, int *first, int *tokens) {
  const long long lo = min(max((long long)a.lists.pos[row], 0ll), a.lists.nnz), hi = min(max((long long)a.lists.pos[row + 1], lo), a.lists.nnz);
  *first = (int)lo;
  *tokens = a.pages > 0 ? (int)max(0ll, min((long long)a.lists.tokens[row], (hi - lo) << a.page_log2)) : 0;
}

// Of a window: how many first tokens count that lie before it, where it starts, and tokens that count in all.  They are numbered in order.
struct Window {
  int sinks, first, count;
  __device__ __forceinline__ int token(int x) const { return x < sinks ? x : (int)((unsigned)first + (unsigned)(x - sinks)); }
};
__device__ __forceinline__ Window window_of(const PagedArgs &a, int seq) {
  // The window goes back from the sequence's own last token, whether the table holds it or not.
  const int length = max(a.windows.lengths[seq], 0), held = a.pages > 0 ? (int)min((long long)length, a.windows.table_width << a.page_log2) : 0;
  Window w;
  w.first = min(max(0, length - a.windows.window), held);
  w.sinks = min(a.windows.sink, w.first);
  w.count = w.sinks + (held - w.first);
  return w;
}

// Lists are cut into units of `chunk` pages.  Unit numbers start at pos[row] / chunk + row for each list, which leaves it at
// least the units it needs, so they are known without a sum over the lists before; those left over do nothing.
__device__ __forceinline__ long long unit_start(const PagedArgs &a, long long row) {
  return min(max((long long)a.lists.pos[row], 0ll), a.lists.nnz) / a.chunk + row;
}

// The list that unit u belongs to (the last one that starts at or before it): 64 candidates a step.
__device__ __forceinline__ int list_of_unit(const PagedArgs &a, int u, int lane) {
  int lo = 0, n = a.lists.rows;
  while (n > 1) {
    const int step = (n + 63) / 64, at = lo + lane * step;
    const unsigned long long before = __ballot(lane * step < n && unit_start(a, at) <= u);
    // positions that do not ascend may give any pattern: the highest candidate at or before u, or the first
    const int pick = before ? 63 - __clzll(before) : 0;
    lo += pick * step;
    n = min(step, n - pick * step);
  }
  return lo;
}

// Eight e4m3 codes as eight numbers of a 16-bit type: exact, times a power of two: exact but for float16's subnormal numbers, and
// those are rounded once, to nearest even.
template <typename T>
__device__ __forceinline__ vec8<T> codes_to(v2i x, float by = 1.0f) {
  v4u r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (std::is_same<T, Bf16>::value) {
      r[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[i], by, false));
      r[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[i], by, true));
    } else {
      r[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[i], by, false));
      r[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)x[i], by, true));
    }
  }
  return __builtin_bit_cast(vec8<T>, r);
}

// Eight 4-bit codes times their scale, as numbers of a 16-bit type (codes and scales have values of their own there but for
// float16's subnormal numbers, where they are rounded once).
template <typename T>
__device__ __forceinline__ vec8<T> codes_to(unsigned x, float by) {
  v4u r;
  if constexpr (std::is_same<T, Bf16>::value) {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, by, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, by, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, by, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, by, 3));
  } else {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, by, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, by, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, by, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, by, 3));
  }
  return __builtin_bit_cast(vec8<T>, r);
}

__device__ __forceinline__ float power_of_two(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0x7f800000u); }

// A unit: up to 16 heads of a group against a stretch of a list.  Its four wavefronts take tiles of 32 tokens in turn, each by
// itself; their maxima, sums and results are joined through LDS.
//   S^T = K Q^T (16x16x32, a head per lane): K goes from memory into the operand's registers, each lane a piece of one token.
//   O^T = V^T P^T: P^T stays in its registers, rounded to the queries' type as a product's operands are, V goes through LDS, where it is read by columns.
// The next tile is loaded into the same registers as soon as they have been used, so all but the first products of a tile
// run under its successor's loads; eight wavefronts a compute unit have 64 KB (8-bit cache) to 128 KB on their way.
// 8-bit codes are multiplied as they are (exact in 16 bits); a key's scale multiplies its score, a value's scale its weight.  With
// float16 only the scale's mantissa does: a weight times a whole scale would leave its range, and in units of the largest scale one large row
// of little weight would push all others' weights below it.  The scale's power of two goes to the value's codes, in units of 2^-7 of the
// largest so far: exact for scales down to 2^-22 of that one, rounded to multiples of 2^-24 units below.
// Bound by memory: 64 sequences of up to 8192 tokens, 32 heads over 8, dim 128, 8-bit cache: 153 us at 4.5 TB/s (a large copy
// reaches 4.75), 160 with float16 queries; one sequence of 16 384 tokens, bf16: 22.4 us, 16.9 of them here (4.0 TB/s) and 5.4 for the join.
// 4-bit codes become 16-bit operands by one conversion with their scale (exact, in float16 down to its subnormal numbers: two bits of mantissa times a power of two), K in registers and V on
// its way into LDS; 128 registers, four workgroups a compute unit, as a row is 64 bytes and its 32 elements a lane one load.  64 sequences of up to 8192
// tokens: 86 us with the join, 78 of them here (4.5 TB/s); one of 16 384: 14.4, 9.6 here (launch, look-ups and two tiles one after the other) and 4.6.
// Windows number their tokens first ones first, so that a unit may hold the end of those and the start of the others; table entries are asked for as
// those of lists are.  128 sequences, window 4096 and 64 first tokens, 4 bits: 133 us, 119 of them here (4.8 TB/s); 4 sequences, bf16: 21.0, 17.0 here (4.0 TB/s).
template <typename T, int CODES, int DP, bool WINDOW>
__global__ __launch_bounds__(256, DP > 128 ? 1 : CODES == kF4 ? 4 : CODES == kF8 ? 3 : 2) void paged_kernel(PagedArgs a) {
  typedef typename T::elem elem;
  constexpr bool F8 = CODES == kF8, F4 = CODES == kF4;
  typedef typename std::conditional<F8, v2i, typename std::conditional<F4, unsigned, v4i>::type>::type raw;  // eight elements
  typedef typename std::conditional<F4, v4u, raw>::type raw_v;                                                // what a lane loads of V at once
  constexpr int KS = DP / 32, DT = DP / 16, PIECES = DP / 8, WIDTH = F8 ? 1 : 2;
  constexpr int V_PIECES = F4 ? DP / 32 : PIECES, RP = 64 / V_PIECES, PASSES = 32 / RP;
  constexpr bool SCALED = F8 && std::is_same<T, F16>::value;
  struct Tokens {
    long long at[32];     // element offsets of the tile's rows
    float ks[F4 ? 4 : 32], vs[F4 ? 4 : 32]; // SCALED: vs holds mantissas, and vp powers of two, those of a lane's rows side by side
    float vp[SCALED ? 32 : 4];
    long long scale_at[F4 ? 32 : 2];
  };
  union Own {  // of a wavefront
    elem v[32 * DP];
    float out[16][DP + 4];
  };
  __shared__ __attribute__((aligned(16))) Own own[4];
  __shared__ __attribute__((aligned(16))) Tokens tokens_of[4][2];
  __shared__ float top[4][16], total[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quarter = lane >> 4;
  unsigned block = xcd_contiguous_block(blockIdx.x, gridDim.x);
  const int ht = block % a.head_tiles;
  block /= a.head_tiles;
  int kh = 0;
  if (WINDOW || !a.lists.each) {
    kh = block % a.kv_heads;
    block /= a.kv_heads;
  }
  const int u = block;
  int seq, part, first = 0, count;
  Window w = {};
  if constexpr (WINDOW) {
    seq = u / a.windows.units_each;
    part = u - seq * a.windows.units_each;
    w = window_of(a, seq);
    count = w.count;
  } else {
    const int row = list_of_unit(a, u, lane);
    seq = a.lists.each ? row / a.kv_heads : row;
    if (a.lists.each) kh = row - seq * a.kv_heads;
    list_of(a, row, &first, &count);
    part = (int)(u - unit_start(a, row));
  }
  const int chunk = WINDOW ? a.chunk : a.chunk << a.page_log2;
  const long long from_l = (long long)part * chunk;
  if (part < 0 || (from_l >= count && part != 0)) return;  // a unit number left over (a list without tokens still writes its zeros)
  const int from = (int)from_l, n = min(chunk, count - from), tiles = (n + 31) / 32;
  const int head0 = kh * a.group + ht * 16, heads = min(16, a.group - ht * 16);

  // Element j of step s of this lane's operands stands for dimension 32 s + 8 quarter + j; with 4-bit codes for DP / 4 quarter + 8 s + j, so
  // that a lane's part of a row is what one load brings (dim 128: 32 elements and their scale).
  const auto dim_of = [&](int s) { return F4 ? DP / 4 * quarter + 8 * s : 32 * s + 8 * quarter; };
  vec8<T> qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = dim_of(s);
    qf[s] = vec8<T>{};
    if (col < heads && d < a.dim) qf[s] = *(const vec8<T> *)((const elem *)a.q + seq * a.q_stride[0] + (head0 + col) * a.q_stride[1] + d);
  }
  const float c = a.scale * 1.4426950408889634f;

  Own &mine = own[wave];
  int page = -1;  // of token `lane & 31` of the tile after the one being loaded
  const auto page_of = [&](int t) {
    const int x = t * 32 + (lane & 31);
    page = -1;
    if (t < tiles && x < n) {
      if constexpr (WINDOW) page = a.windows.table[seq * a.windows.table_width + (w.token(from + x) >> a.page_log2)];
      else page = a.lists.crd[first + ((from + x) >> a.page_log2)];
    }
  };
  unsigned there_next = 0;
  const auto put_tokens = [&](int t) {  // pages into places of rows, for lanes 0 .. 31
    Tokens &x = tokens_of[wave][(t / 4) & 1];
    const bool there = (unsigned)page < (unsigned long long)a.pages;
    there_next = (unsigned)__ballot(there);
    const int number = from + t * 32 + (lane & 31), in = (WINDOW ? w.token(number) : number) & ((1 << a.page_log2) - 1);
    if (lane < 32) {
      x.at[lane] = there ? page * a.stride[0] + kh * a.stride[1] + in * a.stride[2] : 0;
      if (CODES != kNoCodes) {
        const long long s = there ? page * a.scale_stride[0] + kh * a.scale_stride[1] + in * a.scale_stride[2] : 0;
        if constexpr (F4) {
          x.scale_at[lane] = s;
        } else {
          x.ks[lane] = there ? ((const float *)a.k_scale)[s] : 0.f;
          const float vs = there ? ((const float *)a.v_scale)[s] : 0.f;
          x.vs[lane] = SCALED ? 2.f * __builtin_amdgcn_frexp_mantf(vs) : vs;  // (of an infinity or NaN: itself, and its power is infinite)
          if (SCALED) x.vp[lane % RP * PASSES + lane / RP] = power_of_two(vs);
        }
      }
    }
    wave_lds_sync();
  };
  raw kr[2][KS];
  raw_v vr[PASSES];
  constexpr int K_SCALES = DP > 128 ? 2 : 1;  // of a lane's part of a row in 4 bits
  unsigned kb[F4 ? 2 : 1][K_SCALES], vb[F4 ? PASSES : 1];
  const auto load = [&](int t) {
    const Tokens &x = tokens_of[wave][(t / 4) & 1];
    if constexpr (F4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const char *k = a.k + x.at[16 * i + col] / 2;
        const unsigned char *scales = (const unsigned char *)a.k_scale + x.scale_at[16 * i + col];
#pragma unroll
        for (int g = 0; g < K_SCALES; ++g) {  // 32 elements at a time (dim 64: 16)
          const int d = DP / 4 * quarter + 32 * g;
          const bool inside = d < a.dim;
          const char *from = k + (inside ? d / 2 : 0);
          kb[i][g] = scales[inside ? d / 32 : 0];
          if constexpr (DP == 64) {
            const v2u two = *(const v2u *)from;
            kr[i][0] = two[0], kr[i][1] = two[1];
          } else {
            const v4u four = *(const v4u *)from;
#pragma unroll
            for (int s = 0; s < 4; ++s) kr[i][4 * g + s] = four[s];
          }
          if (!inside) kb[i][g] = 127;
#pragma unroll
          for (int s = 0; s < KS / K_SCALES; ++s)
            if (!inside) kr[i][KS / K_SCALES * g + s] = 0;
        }
      }
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int d = (lane % V_PIECES) * 32, row = p * RP + lane / V_PIECES;
        const bool inside = d < a.dim;
        vr[p] = *(const raw_v *)(a.v + (x.at[row] + (inside ? d : 0)) / 2);
        vb[p] = ((const unsigned char *)a.v_scale)[x.scale_at[row] + (inside ? d / 32 : 0)];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const char *k = a.k + x.at[16 * i + col] * WIDTH;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int d = 32 * s + 8 * quarter;
          kr[i][s] = *(const raw *)(k + (d < a.dim ? d : 0) * WIDTH);
          if (a.dim < 32 * s + 32 && d >= a.dim) kr[i][s] = raw{};
        }
      }
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int d = (lane % PIECES) * 8;
        vr[p] = *(const raw_v *)(a.v + (x.at[p * RP + lane / PIECES] + (d < a.dim ? d : 0)) * WIDTH);
      }
    }
  };

  v4f acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  float unit = 0x1p-126f;  // what acc is counted in, a power of two (SCALED)
  page_of(wave);
  put_tokens(wave);
  unsigned there = there_next;
  if (wave < tiles) load(wave);
  page_of(wave + 4);
  for (int t = wave; t < tiles; t += 4) {
    const Tokens &tok = tokens_of[wave][(t / 4) & 1];
    v4f s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        vec8<T> k;
        if constexpr (F8) k = codes_to<T>(kr[i][x]);
        else if constexpr (F4) k = codes_to<T>(kr[i][x], scale_of_byte(kb[i][x / (KS / K_SCALES)]));
        else k = __builtin_bit_cast(vec8<T>, kr[i][x]);
        s[i] = mfma16(k, qf[x], s[i]);
      }
    }
    float unit_to = unit, per_unit = 1.f;
    if constexpr (SCALED) {
      const float most = rows_max(__builtin_bit_cast(float, group_max<16>(__builtin_bit_cast(unsigned, tok.vp[lane & 31]))));
      unit_to = fmaxf(unit, most * 0x1p-7f);
      per_unit = __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(unsigned, unit_to));
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int r = p * RP + lane / V_PIECES, piece = lane % V_PIECES;
      const auto put = [&](int at, vec8<T> v) {
        if (there != 0xffffffffu && !(there >> r & 1)) v = vec8<T>{};  // whatever an unused slot holds: 0 times it must be 0
        *(vec8<T> *)(mine.v + r * DP + ((at ^ turn16<DP>(r)) * 8)) = v;
      };
      if constexpr (F4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) put(4 * piece + i, codes_to<T>(vr[p][i], scale_of_byte(vb[p])));
      } else if constexpr (SCALED) {
        put(piece, codes_to<T>(vr[p], tok.vp[lane / PIECES * PASSES + p] * per_unit));
      } else if constexpr (F8) {
        put(piece, codes_to<T>(vr[p]));
      } else {
        put(piece, __builtin_bit_cast(vec8<T>, vr[p]));
      }
    }
    const unsigned now = there;
    put_tokens(t + 4);
    there = there_next;
    if (t + 4 < tiles) load(t + 4);
    page_of(t + 8);

    float ks[8], vs[8];
    if constexpr (F8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const v4f k4 = *(const v4f *)(tok.ks + 16 * i + 4 * quarter), v4 = *(const v4f *)(tok.vs + 16 * i + 4 * quarter);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ks[4 * i + e] = k4[e];
          vs[4 * i + e] = v4[e];
        }
      }
    }

    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = s[i][e] * (F8 ? c * ks[4 * i + e] : c);
        if (now != 0xffffffffu && !(now >> (16 * i + 4 * quarter + e) & 1)) x = -INFINITY;
        s[i][e] = x;
        best = fmaxf(best, x);
      }
    best = rows_max(best);
    // the maximum in use moves only when it is left behind by more than 2^8
    if (__any(best > m + 8.f) || unit_to != unit) {
      const float to = fmaxf(m, best), keep = to == m ? 1.f : __builtin_amdgcn_exp2f(m - to);
      const float by = SCALED ? keep * (unit * per_unit) : keep;
      m = to;
      l *= keep;
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] *= by;
      unit = unit_to;
    }
    const float off = m == -INFINITY ? 0.f : m;
    vec8<T> pf;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(s[i][e] - off);
        l += p;
        pf[4 * i + e] = (elem)(F8 ? p * vs[4 * i + e] : p);
      }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const int r = 4 * quarter + (col >> 2), d = 16 * i + 4 * (col & 3);
      const elem *p = mine.v + r * DP + ((d >> 3) ^ turn16<DP>(r)) * 8 + (d & 7);  // row + 16 has the same order of pieces
      acc[i] = mfma16(join<T>(read_columns<T>(p), read_columns<T>(p + 16 * DP)), pf, acc[i]);
    }
    wave_lds_sync();
  }
  l = rows_sum(l);
  if (SCALED) {
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] *= unit;
  }
  if (quarter == 0) top[wave][col] = m, total[wave][col] = l;
#pragma unroll
  for (int i = 0; i < DT; ++i) *(v4f *)(&mine.out[col][16 * i + 4 * quarter]) = acc[i];
  __syncthreads();

  const bool whole = count <= chunk;
  const long long unit_id = (long long)(!WINDOW && a.lists.each ? u : u * a.kv_heads + kh) * a.head_tiles + ht;
  for (int x = tid; x < 16 * PIECES; x += 256) {
    const int h = x / PIECES, d = (x % PIECES) * 8;
    if (h >= heads || d >= a.dim) continue;
    float most = top[0][h], sum = 0.f, o[8] = {};
#pragma unroll
    for (int w = 1; w < 4; ++w) most = fmaxf(most, top[w][h]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float by = top[w][h] == most ? 1.f : __builtin_amdgcn_exp2f(top[w][h] - most);
      sum += by * total[w][h];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += by * own[w].out[h][d + e];
    }
    if (whole) {
      const float by = 1.f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = sum == 0.f ? 0.f : o[e] * by;
      *(vec8<T> *)((elem *)a.out + seq * a.out_stride[0] + (head0 + h) * a.out_stride[1] + d) = narrow<T>(o);
      if (a.lse && d == 0)
        a.lse[(long long)seq * a.heads + head0 + h] = sum == 0.f ? -INFINITY : (most + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
    } else {
      float *to = a.partial + (unit_id * 16 + h) * DP + d;
      *(v4f *)to = v4f{o[0], o[1], o[2], o[3]};
      *(v4f *)(to + 4) = v4f{o[4], o[5], o[6], o[7]};
      if (d == 0) *(v2f *)(a.sums + (unit_id * 16 + h) * 2) = v2f{most, sum};
    }
  }
}

// Lists of several units: one workgroup per (sequence, head), 64 units at a time, a quarter of them to each wavefront and
// four of those on their way (one after the other they took 45 us for 64 units); always in the same order.
template <typename T, int DP, bool WINDOW>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  typedef typename T::elem elem;
  constexpr int E = DP / 64;
  typedef float vec __attribute__((ext_vector_type(E)));
  __shared__ float factor[64];
  __shared__ __attribute__((aligned(16))) float part[3][DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seq = blockIdx.y, head = blockIdx.x, kh = head / a.group, in = head - kh * a.group;
  const long long row = !WINDOW && a.lists.each ? (long long)seq * a.kv_heads + kh : seq;
  int first, count;
  if constexpr (WINDOW) count = window_of(a, seq).count;
  else list_of(a, row, &first, &count);
  const int chunk = WINDOW ? a.chunk : a.chunk << a.page_log2, needed = (int)(((long long)count + chunk - 1) / chunk);
  if (needed <= 1) return;
  const long long u0 = WINDOW ? row * a.windows.units_each : unit_start(a, row);
  const int units = (int)min((long long)needed, a.units - u0);  // fewer only where positions descend
  const auto id = [&](int x) { return ((!WINDOW && a.lists.each ? u0 + x : (u0 + x) * a.kv_heads + kh) * a.head_tiles + in / 16) * 16 + in % 16; };
  float most = -INFINITY;
  for (int x = lane; x < units; x += 64) most = fmaxf(most, a.sums[id(x) * 2]);
  for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
  float sum = 0.f, o[E] = {};
  for (int x0 = 0; x0 < units; x0 += 64) {
    float by = 0.f, s1 = 0.f;
    if (x0 + lane < units) {
      const v2f s = *(const v2f *)(a.sums + id(x0 + lane) * 2);
      by = s[0] == most ? 1.f : __builtin_amdgcn_exp2f(s[0] - most);
      s1 = s[1];
    }
    sum += group_sum<64>(by * s1);
    __syncthreads();
    if (wave == 0) factor[lane] = by;
    __syncthreads();
    const int n = min(64, units - x0);
    for (int x = wave; x < n; x += 16) {
      vec f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = *(const vec *)(a.partial + id(x0 + min(x + 4 * i, n - 1)) * DP + lane * E);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = x + 4 * i < n ? factor[x + 4 * i] : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += x + 4 * i < n ? w * f[i][e] : 0.f;
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave - 1][lane * E + e] = o[e];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E + e;
    o[e] += part[0][d];
    o[e] += part[1][d];
    o[e] += part[2][d];
    if (d < a.dim) ((elem *)a.out)[seq * a.out_stride[0] + head * a.out_stride[1] + d] = (elem)(sum == 0.f ? 0.f : o[e] / sum);
  }
  if (a.lse && lane == 0) a.lse[(long long)seq * a.heads + head] = sum == 0.f ? -INFINITY : (most + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// Whether some sequence may have several units, whose results are joined.
bool several_units(const PagedArgs &a) { return a.windowed ? a.windows.units_each > 1 : a.lists.nnz > a.chunk; }

template <typename T, int CODES, int DP, bool WINDOW>
int launch_paged(const PagedArgs &a, hipStream_t st) {
  const long long blocks = (long long)a.units * (!WINDOW && a.lists.each ? 1 : a.kv_heads) * a.head_tiles;
  LAPIS_REQUIRE(blocks * 256 < (INT64_C(1) << 32), "paged_attention: %lld units of work", blocks);
  hipLaunchKernelGGL((paged_kernel<T, CODES, DP, WINDOW>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  LAPIS_LAUNCH_CHECK();
  if (several_units(a)) {
    hipLaunchKernelGGL((paged_join_kernel<T, DP, WINDOW>), dim3((unsigned)a.heads, (unsigned)a.seqs), dim3(256), 0, st, a);
    LAPIS_LAUNCH_CHECK();
  }
  return LAPIS_HIP_OK;
}

template <bool WINDOW>
int launch_paged(const PagedArgs &a, int dtype, int cache_dtype, hipStream_t st) {
  const auto with = [&](auto type, auto codes) {
    typedef decltype(type) T;
    constexpr int CODES = decltype(codes)::value;
    return a.dim <= 64 ? launch_paged<T, CODES, 64, WINDOW>(a, st) : a.dim <= 128 ? launch_paged<T, CODES, 128, WINDOW>(a, st) : launch_paged<T, CODES, 256, WINDOW>(a, st);
  };
  const auto of = [&](auto type) {
    switch (codes_of(cache_dtype)) {
      case kF4: return with(type, std::integral_constant<int, kF4>());
      case kF8: return with(type, std::integral_constant<int, kF8>());
      default: return with(type, std::integral_constant<int, kNoCodes>());
    }
  };
  return dtype == LAPIS_HIP_BF16 ? of(Bf16()) : of(F16());
}

// What calls over lists and over windows have alike.
int read_paged(const char *what, const lapis_hip_kv_cache *c, int64_t seqs, int64_t heads, int dtype, const lapis_hip_rows &q, const lapis_hip_rows &out,
               float *lse, float scale, PagedArgs *a) {
  LAPIS_REQUIRE(seqs >= 0 && seqs <= 65535 && heads >= 0 && heads <= 65535 && heads % c->heads == 0,
                "%s: %lld sequences and %lld heads over a cache of %d", what, (long long)seqs, (long long)heads, c->heads);
  LAPIS_REQUIRE(is_16bit(dtype) && (c->dtype == dtype || codes_of(c->dtype) != kNoCodes), "%s: queries of type %d and a cache of type %d", what, dtype, c->dtype);
  *a = {};
  a->q = static_cast<const char *>(q.data);
  a->out = static_cast<char *>(out.data);
  for (int i = 0; i < 2; ++i) a->q_stride[i] = q.stride[2 * i], a->out_stride[i] = out.stride[2 * i];
  a->k = static_cast<const char *>(c->k);
  a->v = static_cast<const char *>(c->v);
  a->k_scale = c->k_scale;
  a->v_scale = c->v_scale;
  for (int i = 0; i < 3; ++i) a->stride[i] = c->stride[i], a->scale_stride[i] = c->scale_stride[i];
  a->pages = c->pages;
  a->seqs = (int)seqs;
  a->heads = (int)heads;
  a->kv_heads = c->heads;
  a->dim = c->dim;
  a->page_log2 = __builtin_ctz((unsigned)c->page);
  a->lse = lse;
  a->scale = scale;
  a->group = a->heads / c->heads;
  a->head_tiles = (int)ceil_div(std::max(a->group, 1), 16);
  return LAPIS_HIP_OK;
}

int read_paged(const char *what, const lapis_hip_kv_cache *c, const lapis_hip_paged_args *p, PagedArgs *a) {
  int rc = check_cache(what, c);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  rc = read_paged(what, c, p->seqs, p->heads, p->dtype, p->q, p->out, p->lse, p->scale, a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p->lists == p->seqs || p->lists == p->seqs * c->heads, "%s: %lld lists of pages for %lld sequences", what,
                (long long)p->lists, (long long)p->seqs);
  LAPIS_REQUIRE(p->nnz >= 0 && p->nnz <= INT32_MAX && p->nnz * c->page <= INT32_MAX, "%s: %lld pages listed", what, (long long)p->nnz);
  LAPIS_REQUIRE(p->lists <= INT32_MAX, "%s: %lld lists", what, (long long)p->lists);
  a->lists.nnz = p->nnz;
  a->lists.each = p->lists != p->seqs;
  a->lists.pos = p->pos;
  a->lists.crd = p->crd;
  a->lists.tokens = p->tokens;
  a->lists.rows = (int)p->lists;
  // Units for two workgroups a compute unit, of 128 to 1024 tokens: shorter ones cost more than they spread (a partial result
  // and its join), longer ones leave compute units waiting for the last.  Two of them too where three (8 bits) or four (4 bits) fit a compute unit: one sequence
  // of 16 384 tokens, 32 heads over 8, dim 128, 4 bits 14.2 us, for four 17.4; 64 of 8192 123.9 and 123.7; 8 bits, for two and three: 18.2 and 21.3, 223 and 223.
  const int64_t copies = (int64_t)a->head_tiles * (a->lists.each ? 1 : c->heads), wanted = std::max(2 * device_cu_count(), 1);
  const int64_t tokens = std::min<int64_t>(std::max<int64_t>(p->nnz * c->page * copies / wanted, 128), 1024);
  a->chunk = (int)std::max<int64_t>(tokens / c->page, 1);
  const int64_t units = p->nnz / a->chunk + p->lists;
  LAPIS_REQUIRE(units <= INT32_MAX, "%s: %lld units of work", what, (long long)units);
  a->units = (int)units;
  return LAPIS_HIP_OK;
}

int read_window(const char *what, const lapis_hip_kv_cache *c, const lapis_hip_paged_window_args *p, PagedArgs *a) {
  int rc = check_cache(what, c);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  rc = read_paged(what, c, p->seqs, p->heads, p->dtype, p->q, p->out, p->lse, p->scale, a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p->window >= 1 && p->sink >= 0, "%s: a window of %lld and the first %lld tokens", what, (long long)p->window, (long long)p->sink);
  LAPIS_REQUIRE(p->table_width >= 0 && p->table_width <= INT32_MAX / c->page, "%s: a table of %lld pages", what, (long long)p->table_width);
  a->windowed = true;
  a->windows.table = p->table;
  a->windows.lengths = p->lengths;
  a->windows.table_width = p->table_width;
  const int64_t longest = p->table_width * c->page;
  a->windows.window = (int)std::min<int64_t>(p->window, INT32_MAX);
  a->windows.sink = (int)std::min<int64_t>(p->sink, INT32_MAX);
  // Tokens that count in a sequence, at most; units as above, but no more than four a compute unit for any one sequence: every sequence has as many, whatever
  // its length, and a partial result for each.  A table of 2^20 tokens, 8 key-value heads, dim 128, 16 and 4 bits, units of 1024 tokens always and so: 64
  // sequences of 8192, 752 us, 404 and 4.4 GB of scratch memory, and 425, 188 and 0.5 GB; one of them of 2^20, 3935 and 1607 us, and 3545 and 1216; a
  // single one of 2^20, 770 and 284, and 719 and 228.
  const int64_t most = std::min(longest, std::min(p->window, longest) + std::min(p->sink, longest));
  const int64_t copies = std::min<int64_t>((int64_t)a->head_tiles * c->heads, 65535), wanted = std::max(2 * device_cu_count(), 1);  // (a cache may have more heads than that, a call with queries not)
  const int64_t longest_unit = std::min<int64_t>(std::max<int64_t>(1024, most * copies / (2 * wanted)), 1 << 30);
  a->chunk = (int)(std::min<int64_t>(std::max<int64_t>(p->seqs * most * copies / wanted, 128), longest_unit) / 32 * 32);
  a->windows.units_each = (int)std::max<int64_t>(1, ceil_div(most, a->chunk));
  const int64_t units = p->seqs * a->windows.units_each;
  LAPIS_REQUIRE(units <= INT32_MAX, "%s: %lld units of work", what, (long long)units);
  a->units = (int)units;
  return LAPIS_HIP_OK;
}

// bytes of the partial results, and where the sums lie behind them
int64_t partial_bytes(const PagedArgs &a, int64_t *sums_at) {
  const int dp = a.dim <= 64 ? 64 : a.dim <= 128 ? 128 : 256;
  const int64_t ids = (int64_t)a.units * (!a.windowed && a.lists.each ? 1 : a.kv_heads) * a.head_tiles * 16;
  *sums_at = ids * dp * 4;
  return several_units(a) ? ids * (dp + 2) * 4 : 0;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

namespace {

int paged_work(const PagedArgs &a, const char *what, int64_t *bytes) {
  LAPIS_REQUIRE(bytes, "%s: null result", what);
  int64_t sums_at;
  *bytes = partial_bytes(a, &sums_at);
  return LAPIS_HIP_OK;
}

int check_rows(const PagedArgs &a, const char *what, const lapis_hip_rows &q, const lapis_hip_rows &out) {
  LAPIS_REQUIRE(aligned16(a.q) && aligned16(a.out) && strides_of_8(q.stride, 3) && strides_of_8(out.stride, 3),
                "%s: queries or results that are not on 16-byte boundaries or strides that are no multiples of 8", what);
  return LAPIS_HIP_OK;
}

int give_work(PagedArgs &a, const char *what, void *work) {
  int64_t sums_at;
  if (partial_bytes(a, &sums_at) == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(work && aligned16(work), "%s: work that is null or not on a 16-byte boundary", what);
  a.partial = static_cast<float *>(work);
  a.sums = reinterpret_cast<float *>(static_cast<char *>(work) + sums_at);
  return LAPIS_HIP_OK;
}

}  // namespace

extern "C" int lapis_hip_paged_attention_work(const lapis_hip_kv_cache *cache, const lapis_hip_paged_args *args, int64_t *bytes) {
  PagedArgs a;
  const int rc = read_paged("paged_attention", cache, args, &a);
  return rc != LAPIS_HIP_OK ? rc : paged_work(a, "paged_attention", bytes);
}

extern "C" int lapis_hip_paged_attention(const lapis_hip_kv_cache *cache, const lapis_hip_paged_args *args, lapis_hip_stream_t stream) {
  PagedArgs a;
  int rc = read_paged("paged_attention", cache, args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.seqs == 0 || a.heads == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(a.q && a.out && a.lists.pos && a.lists.tokens && (a.lists.crd || a.lists.nnz == 0), "paged_attention: null operands");
  rc = check_rows(a, "paged_attention", args->q, args->out);
  if (rc == LAPIS_HIP_OK) rc = give_work(a, "paged_attention", args->work);
  return rc != LAPIS_HIP_OK ? rc : launch_paged<false>(a, args->dtype, cache->dtype, as_stream(stream));
}

extern "C" int lapis_hip_paged_window_attention_work(const lapis_hip_kv_cache *cache, const lapis_hip_paged_window_args *args, int64_t *bytes) {
  PagedArgs a;
  const int rc = read_window("paged_window_attention", cache, args, &a);
  return rc != LAPIS_HIP_OK ? rc : paged_work(a, "paged_window_attention", bytes);
}

extern "C" int lapis_hip_paged_window_attention(const lapis_hip_kv_cache *cache, const lapis_hip_paged_window_args *args, lapis_hip_stream_t stream) {
  PagedArgs a;
  int rc = read_window("paged_window_attention", cache, args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.seqs == 0 || a.heads == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(a.q && a.out && a.windows.lengths && (a.windows.table || a.windows.table_width == 0), "paged_window_attention: null operands");
  rc = check_rows(a, "paged_window_attention", args->q, args->out);
  if (rc == LAPIS_HIP_OK) rc = give_work(a, "paged_window_attention", args->work);
  return rc != LAPIS_HIP_OK ? rc : launch_paged<true>(a, args->dtype, cache->dtype, as_stream(stream));
}
