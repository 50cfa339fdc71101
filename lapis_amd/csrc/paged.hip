// Attention of one new token of each sequence over the pages of a cache that a CSR row lists.
#include "mfma.hpp"

namespace lapis {
namespace {

struct PagedArgs {
  const char *q;
  char *out;
  long long q_stride[2], out_stride[2];
  const char *k, *v;
  const float *k_scale, *v_scale;
  long long stride[3], scale_stride[3];
  long long pages, nnz;
  int seqs, lists, heads, kv_heads, group, dim, page_log2;
  bool each;  // a list per key-value head
  const int *pos, *crd, *tokens;
  float *lse;
  float scale;
  int chunk, units, head_tiles;  // pages a unit, units of all lists, tiles of 16 heads
  float *partial, *sums;         // of each unit: 16 x DP, and 16 maxima and sums
};

// Pages that a row lists and tokens that count in them, whatever pos and tokens hold.
__device__ __forceinline__ void list_of(const PagedArgs &a, long long row, int *first, int *tokens) {
  const long long lo = min(max((long long)a.pos[row], 0ll), a.nnz), hi = min(max((long long)a.pos[row + 1], lo), a.nnz);
  *first = (int)lo;
  *tokens = a.pages > 0 ? (int)max(0ll, min((long long)a.tokens[row], (hi - lo) << a.page_log2)) : 0;
}

// Lists are cut into units of `chunk` pages.  Unit numbers start at pos[row] / chunk + row for each list, which leaves it at
// least the units it needs, so they are known without a sum over the lists before; those left over do nothing.
__device__ __forceinline__ long long unit_start(const PagedArgs &a, long long row) {
  return min(max((long long)a.pos[row], 0ll), a.nnz) / a.chunk + row;
}

// The list that unit u belongs to (the last one that starts at or before it): 64 candidates a step.
__device__ __forceinline__ int list_of_unit(const PagedArgs &a, int u, int lane) {
  int lo = 0, n = a.lists;
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

__device__ __forceinline__ float power_of_two(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0x7f800000u); }

// A unit: up to 16 heads of a group against a stretch of a list.  Its four wavefronts take tiles of 32 tokens in turn, each by
// itself; their maxima, sums and results are joined through LDS.
//   S^T = K Q^T (16x16x32, a head per lane): K goes from memory into the operand's registers, each lane a piece of one token.
//   O^T = V^T P^T: P^T stays in its registers, V goes through LDS, where it is read by columns.
// The next tile is loaded into the same registers as soon as they have been used, so all but the first products of a tile
// run under its successor's loads; eight wavefronts a compute unit have 64 KB (8-bit cache) to 128 KB on their way.
// 8-bit codes are multiplied as they are (exact in 16 bits); a key's scale multiplies its score, a value's scale its weight.  With
// float16 only the scale's mantissa does: a weight times a whole scale would leave its range, and in units of the largest scale one large row
// of little weight would push all others' weights below it.  The scale's power of two goes to the value's codes, in units of 2^-7 of the
// largest so far: exact for scales down to 2^-22 of that one, rounded to multiples of 2^-24 units below.
// Bound by memory: 64 sequences of up to 8192 tokens, 32 heads over 8, dim 128, 8-bit cache: 153 us at 4.5 TB/s (a large copy
// reaches 4.75), 160 with float16 queries; one sequence of 16 384 tokens, bf16: 22.4 us, 16.9 of them here (4.0 TB/s) and 5.4 for the join.
template <typename T, bool F8, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : F8 ? 3 : 2) void paged_kernel(PagedArgs a) {
  typedef typename T::elem elem;
  typedef typename std::conditional<F8, v2i, v4i>::type raw;  // eight elements
  constexpr int KS = DP / 32, DT = DP / 16, PIECES = DP / 8, RP = 64 / PIECES, PASSES = 32 / RP, WIDTH = F8 ? 1 : 2;
  constexpr bool SCALED = F8 && std::is_same<T, F16>::value;
  struct Tokens {
    long long at[32];     // element offsets of the tile's rows
    float ks[32], vs[32]; // SCALED: vs holds mantissas, and vp powers of two, those of a lane's rows side by side
    float vp[SCALED ? 32 : 4];
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
  if (!a.each) {
    kh = block % a.kv_heads;
    block /= a.kv_heads;
  }
  const int u = block, row = list_of_unit(a, u, lane);
  const int seq = a.each ? row / a.kv_heads : row;
  if (a.each) kh = row - seq * a.kv_heads;
  int first, count;
  list_of(a, row, &first, &count);
  const int part = (int)(u - unit_start(a, row));
  const int chunk = a.chunk << a.page_log2;  // tokens
  const long long from_l = (long long)part * chunk;
  if (part < 0 || (from_l >= count && part != 0)) return;  // a unit number left over (a list without tokens still writes its zeros)
  const int from = (int)from_l, n = min(chunk, count - from), tiles = (n + 31) / 32;
  const int head0 = kh * a.group + ht * 16, heads = min(16, a.group - ht * 16);

  // element j of step s of this lane's operands stands for dimension 32 s + 8 quarter + j
  vec8<T> qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = 32 * s + 8 * quarter;
    qf[s] = vec8<T>{};
    if (col < heads && d < a.dim) qf[s] = *(const vec8<T> *)((const elem *)a.q + seq * a.q_stride[0] + (head0 + col) * a.q_stride[1] + d);
  }
  const float c = a.scale * 1.4426950408889634f;

  Own &mine = own[wave];
  int page = -1;  // of token `lane & 31` of the tile after the one being loaded
  const auto page_of = [&](int t) {
    const int x = t * 32 + (lane & 31);
    page = t < tiles && x < n ? a.crd[first + ((from + x) >> a.page_log2)] : -1;
  };
  unsigned there_next = 0;
  const auto put_tokens = [&](int t) {  // pages into places of rows, for lanes 0 .. 31
    Tokens &x = tokens_of[wave][(t / 4) & 1];
    const bool there = (unsigned)page < (unsigned long long)a.pages;
    there_next = (unsigned)__ballot(there);
    const int in = (from + t * 32 + (lane & 31)) & ((1 << a.page_log2) - 1);
    if (lane < 32) {
      x.at[lane] = there ? page * a.stride[0] + kh * a.stride[1] + in * a.stride[2] : 0;
      if (F8) {
        const long long s = there ? page * a.scale_stride[0] + kh * a.scale_stride[1] + in * a.scale_stride[2] : 0;
        x.ks[lane] = there ? a.k_scale[s] : 0.f;
        const float vs = there ? a.v_scale[s] : 0.f;
        x.vs[lane] = SCALED ? 2.f * __builtin_amdgcn_frexp_mantf(vs) : vs;  // (of an infinity or NaN: itself, and its power is infinite)
        if (SCALED) x.vp[lane % RP * PASSES + lane / RP] = power_of_two(vs);
      }
    }
    wave_lds_sync();
  };
  raw kr[2][KS], vr[PASSES];
  const auto load = [&](int t) {
    const Tokens &x = tokens_of[wave][(t / 4) & 1];
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
      vr[p] = *(const raw *)(a.v + (x.at[p * RP + lane / PIECES] + (d < a.dim ? d : 0)) * WIDTH);
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
      const int r = p * RP + lane / PIECES, piece = lane % PIECES;
      vec8<T> v;
      if constexpr (SCALED) v = codes_to<T>(vr[p], tok.vp[lane / PIECES * PASSES + p] * per_unit);
      else if constexpr (F8) v = codes_to<T>(vr[p]);
      else v = __builtin_bit_cast(vec8<T>, vr[p]);
      if (there != 0xffffffffu && !(there >> r & 1)) v = vec8<T>{};  // whatever an unused slot holds: 0 times it must be 0
      *(vec8<T> *)(mine.v + r * DP + ((piece ^ turn16<DP>(r)) * 8)) = v;
    }
    const unsigned now = there;
    put_tokens(t + 4);
    there = there_next;
    if (t + 4 < tiles) load(t + 4);
    page_of(t + 8);

    float ks[8], vs[8];
    if (F8) {
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
  const long long unit_id = (long long)(a.each ? u : u * a.kv_heads + kh) * a.head_tiles + ht;
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
template <typename T, int DP>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  typedef typename T::elem elem;
  constexpr int E = DP / 64;
  typedef float vec __attribute__((ext_vector_type(E)));
  __shared__ float factor[64];
  __shared__ __attribute__((aligned(16))) float part[3][DP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seq = blockIdx.y, head = blockIdx.x, kh = head / a.group, in = head - kh * a.group;
  const long long row = a.each ? (long long)seq * a.kv_heads + kh : seq;
  int first, count;
  list_of(a, row, &first, &count);
  const int chunk = a.chunk << a.page_log2, needed = (int)(((long long)count + chunk - 1) / chunk);
  if (needed <= 1) return;
  const long long u0 = unit_start(a, row);
  const int units = (int)min((long long)needed, a.units - u0);  // fewer only where positions descend
  const auto id = [&](int x) { return ((a.each ? u0 + x : (u0 + x) * a.kv_heads + kh) * a.head_tiles + in / 16) * 16 + in % 16; };
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

template <typename T, bool F8, int DP>
int launch_paged(const PagedArgs &a, hipStream_t st) {
  const long long blocks = (long long)a.units * (a.each ? 1 : a.kv_heads) * a.head_tiles;
  LAPIS_REQUIRE(blocks * 256 < (INT64_C(1) << 32), "paged_attention: %lld units of work", blocks);
  hipLaunchKernelGGL((paged_kernel<T, F8, DP>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  LAPIS_LAUNCH_CHECK();
  if (a.nnz > a.chunk) {  // some list may have several units
    hipLaunchKernelGGL((paged_join_kernel<T, DP>), dim3((unsigned)a.heads, (unsigned)a.seqs), dim3(256), 0, st, a);
    LAPIS_LAUNCH_CHECK();
  }
  return LAPIS_HIP_OK;
}

template <typename T, bool F8>
int launch_paged(const PagedArgs &a, hipStream_t st) {
  return a.dim <= 64 ? launch_paged<T, F8, 64>(a, st) : a.dim <= 128 ? launch_paged<T, F8, 128>(a, st) : launch_paged<T, F8, 256>(a, st);
}

int read_paged(const char *what, const lapis_hip_kv_cache *c, const lapis_hip_paged_args *p, PagedArgs *a) {
  const int rc = check_cache(what, c);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  LAPIS_REQUIRE(p->seqs >= 0 && p->seqs <= 65535 && p->heads >= 0 && p->heads <= 65535 && p->heads % c->heads == 0,
                "%s: %lld sequences and %lld heads over a cache of %d", what, (long long)p->seqs, (long long)p->heads, c->heads);
  LAPIS_REQUIRE(p->lists == p->seqs || p->lists == p->seqs * c->heads, "%s: %lld lists of pages for %lld sequences", what,
                (long long)p->lists, (long long)p->seqs);
  LAPIS_REQUIRE(p->nnz >= 0 && p->nnz <= INT32_MAX && p->nnz * c->page <= INT32_MAX, "%s: %lld pages listed", what, (long long)p->nnz);
  LAPIS_REQUIRE(p->lists <= INT32_MAX, "%s: %lld lists", what, (long long)p->lists);
  LAPIS_REQUIRE(is_16bit(p->dtype) && (c->dtype == p->dtype || c->dtype == LAPIS_HIP_F8E4M3), "%s: queries of type %d and a cache of type %d",
                what, p->dtype, c->dtype);
  *a = {};
  a->q = static_cast<const char *>(p->q.data);
  a->out = static_cast<char *>(p->out.data);
  for (int i = 0; i < 2; ++i) a->q_stride[i] = p->q.stride[2 * i], a->out_stride[i] = p->out.stride[2 * i];
  a->k = static_cast<const char *>(c->k);
  a->v = static_cast<const char *>(c->v);
  a->k_scale = c->k_scale;
  a->v_scale = c->v_scale;
  for (int i = 0; i < 3; ++i) a->stride[i] = c->stride[i], a->scale_stride[i] = c->scale_stride[i];
  a->pages = c->pages;
  a->nnz = p->nnz;
  a->seqs = (int)p->seqs;
  a->heads = (int)p->heads;
  a->kv_heads = c->heads;
  a->dim = c->dim;
  a->page_log2 = __builtin_ctz((unsigned)c->page);
  a->each = p->lists != p->seqs;
  a->pos = p->pos;
  a->crd = p->crd;
  a->tokens = p->tokens;
  a->lse = p->lse;
  a->scale = p->scale;
  a->lists = (int)p->lists;
  a->group = a->heads / c->heads;
  a->head_tiles = (int)ceil_div(std::max(a->group, 1), 16);
  // Units for two workgroups a compute unit, of 128 to 1024 tokens: shorter ones cost more than they spread (a partial result
  // and its join), longer ones leave compute units waiting for the last.
  const int64_t copies = (int64_t)a->head_tiles * (a->each ? 1 : c->heads), wanted = std::max(2 * device_cu_count(), 1);
  const int64_t tokens = std::min<int64_t>(std::max<int64_t>(p->nnz * c->page * copies / wanted, 128), 1024);
  a->chunk = (int)std::max<int64_t>(tokens / c->page, 1);
  const int64_t units = p->nnz / a->chunk + p->lists;
  LAPIS_REQUIRE(units <= INT32_MAX, "%s: %lld units of work", what, (long long)units);
  a->units = (int)units;
  return LAPIS_HIP_OK;
}

// bytes of the partial results, and where the sums lie behind them
int64_t partial_bytes(const PagedArgs &a, int64_t *sums_at) {
  const int dp = a.dim <= 64 ? 64 : a.dim <= 128 ? 128 : 256;
  const int64_t ids = (int64_t)a.units * (a.each ? 1 : a.kv_heads) * a.head_tiles * 16;
  *sums_at = ids * dp * 4;
  return a.nnz > a.chunk ? ids * (dp + 2) * 4 : 0;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_paged_attention_work(const lapis_hip_kv_cache *cache, const lapis_hip_paged_args *args, int64_t *bytes) {
  PagedArgs a;
  const int rc = read_paged("paged_attention", cache, args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "paged_attention: null result");
  int64_t sums_at;
  *bytes = partial_bytes(a, &sums_at);
  return LAPIS_HIP_OK;
}

extern "C" int lapis_hip_paged_attention(const lapis_hip_kv_cache *cache, const lapis_hip_paged_args *args, lapis_hip_stream_t stream) {
  PagedArgs a;
  const int rc = read_paged("paged_attention", cache, args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.seqs == 0 || a.heads == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(a.q && a.out && a.pos && a.tokens && (a.crd || a.nnz == 0), "paged_attention: null operands");
  LAPIS_REQUIRE(aligned16(a.q) && aligned16(a.out) && strides_of_8(args->q.stride, 3) && strides_of_8(args->out.stride, 3),
                "paged_attention: queries or results that are not on 16-byte boundaries or strides that are no multiples of 8");
  int64_t sums_at;
  if (partial_bytes(a, &sums_at) > 0) {
    LAPIS_REQUIRE(args->work && aligned16(args->work), "paged_attention: work that is null or not on a 16-byte boundary");
    a.partial = static_cast<float *>(args->work);
    a.sums = reinterpret_cast<float *>(static_cast<char *>(args->work) + sums_at);
  }
  const bool f8 = cache->dtype == LAPIS_HIP_F8E4M3, bf16 = args->dtype == LAPIS_HIP_BF16;
  const hipStream_t st = as_stream(stream);
  if (bf16) return f8 ? launch_paged<Bf16, true>(a, st) : launch_paged<Bf16, false>(a, st);
  return f8 ? launch_paged<F16, true>(a, st) : launch_paged<F16, false>(a, st);
}
