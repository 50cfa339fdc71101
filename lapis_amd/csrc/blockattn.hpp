// What the forward and backward kernels of attention over lists of blocks and over windows are given.
#pragma once
#include "mfma.hpp"

namespace lapis {

struct View {
  char *data;
  long long stride[3];  // elements between batch entries, tokens, heads
};

struct BlockArgs {
  View q, k, v, out, dout, dq, dk, dv;
  float *lse;
  const int *pos, *crd;
  long long nnz;
  int batch, queries, keys, heads, kv_heads, group, dim;
  int block_m, block_n_log2, rows, columns;  // rows and columns of a list
  int causal, shift;                         // query i stands at i + shift
  float scale;
  int window, sink;                          // instead of lists: keys behind position - window, and the first ones
};

// Entries of a row of the structure, whatever pos holds.
__device__ __forceinline__ void entries_of(const int *pos, long long nnz, long long row, int *first, int *count) {
  const long long lo = min(max((long long)pos[row], 0ll), nnz), hi = min(max((long long)pos[row + 1], lo), nnz);
  *first = (int)lo;
  *count = (int)(hi - lo);
}
__device__ __forceinline__ void entries_of(const BlockArgs &a, long long row, int *first, int *count) { entries_of(a.pos, a.nnz, row, first, count); }

constexpr int kAbsent = 0x7fff0000;  // first key of sixteen that do not exist

// Keys of a list in the order of its entries, sixteen at a time: blocks hold at least sixteen, so sixteen neighbouring
// places of the list are sixteen neighbouring keys.  (The list has an entry; with blocks listed over and over its places pass 31 bits.)
__device__ __forceinline__ int first_key(const BlockArgs &a, int first, int count, long long place) {
  const long long e = place >> a.block_n_log2;
  const int block = a.crd[first + (int)min(e, count - 1ll)];
  const int key = (int)((unsigned)block << a.block_n_log2) + ((int)place & ((1 << a.block_n_log2) - 1));
  return e < count && (unsigned)block < (unsigned)a.columns ? key : kAbsent;
}

// The keys that queries q0 .. see, `held` of them, over a window: the first ones that lie before it, and from where it starts for the first
// of them to the last one's own.  Sixteen at a time, as those of lists, so that the window starts at a multiple of sixteen and no key
// comes twice.
struct Span {
  int sinks, start, count;  // sixteens of the first keys, first key of the window's, sixteens in all
  __device__ __forceinline__ int first_key(int place16) const {
    return place16 >= count ? kAbsent : place16 < sinks ? 16 * place16 : start + 16 * (place16 - sinks);
  }
};
__device__ __forceinline__ Span span_of(const BlockArgs &a, int q0, int held) {
  const int last = q0 + held - 1 + a.shift;
  Span s = {0, 0, 0};
  if (last < 0) return s;
  s.start = max(0, q0 + a.shift - a.window + 1) & ~15;
  s.sinks = (min(a.sink, s.start) + 15) / 16;
  s.count = s.sinks + (last - s.start) / 16 + 1;
  return s;
}

// Which keys a row sees: up to `limit`, and over a window the last ones of them and the first ones.  (Differences of whole numbers and no || or &&:
// those become branches, a dozen instructions for each key of a tile that wait for one another.  1001 queries behind 2437 keys, window 300, 12 heads: 22.2 us so and 19.9 without.)
template <bool WINDOW>
struct Sight {
  int limit, sinks;
  unsigned window;
  __device__ __forceinline__ Sight(const BlockArgs &a, int limit_) : limit(WINDOW ? max(limit_, -1) : limit_), sinks(min(a.sink, limit + 1)), window((unsigned)a.window) {}
  __device__ __forceinline__ bool sees(int key) const {
    if constexpr (WINDOW) return (int)((unsigned)(limit - key) < window) | (int)(key < sinks);  // (0 <= limit - key < window)
    else return key <= limit;
  }
};

// Tiles of KT keys that a list has.  They are numbered with 31 bits: more would be 2^36 keys of one list, of the 2^30 there are.
template <int KT>
__device__ __forceinline__ int tiles_of(const BlockArgs &a, int count) {
  return a.keys > 0 ? (int)min((((long long)count << a.block_n_log2) + KT - 1) / KT, 0x7fffff00ll) : 0;
}

// Tiles of KT keys and values of a list on their way into two LDS buffers each, a workgroup of NW wavefronts sharing the
// work: sixteen rows at a time lie in one place.  A key that is not there is read from the last one: whoever uses the tile
// gives it no weight, and looks for values that are no numbers wherever a mask cuts.
// WINDOW: the tiles of a span.
template <typename T, int DP, int NW, int KT, bool V_BY_COLUMNS, bool WINDOW = false>
struct KeyTiles {
  typedef typename T::elem elem;
  static constexpr int PIECES = DP / 8, RP = NW * 64 / PIECES, PASSES = KT / RP, CH = KT / 16;
  static_assert(RP % 16 == 0, "a thread has the same row of each sixteen");
  const BlockArgs &a;
  const int first, count, wave, my_row, in16, kd, vd;
  const elem *kp, *vp;
  long long k_off, v_off;
  unsigned k_to, v_to;
  unsigned k_together, v_together;  // bytes from a tile's first row to this thread's part, where its rows lie one behind the other
  bool near;                        // they reach that far
  Span span = {};

  __device__ __forceinline__ KeyTiles(const BlockArgs &a_, int b, int kh, int first_, int count_, int tid, const elem *k_tile, const elem *v_tile)
      : a(a_), first(first_), count(count_), wave(__builtin_amdgcn_readfirstlane(tid >> 6)), my_row(tid / PIECES), in16(my_row & 15),
        kd(((tid % PIECES) ^ turn<DP>(my_row)) * 8), vd(((tid % PIECES) ^ (V_BY_COLUMNS ? column_turn<DP>(my_row) : turn<DP>(my_row))) * 8) {
    kp = (const elem *)a.k.data + b * a.k.stride[0] + kh * a.k.stride[2];
    vp = (const elem *)a.v.data + b * a.v.stride[0] + kh * a.v.stride[2];
    k_off = in16 * a.k.stride[1] + kd;
    v_off = in16 * a.v.stride[1] + vd;
    k_to = lds_address(k_tile) + wave * 1024;
    v_to = lds_address(v_tile) + wave * 1024;
    near = (unsigned long long)a.k.stride[1] < (1u << 26) && (unsigned long long)a.v.stride[1] < (1u << 26);
    k_together = (my_row * (unsigned)a.k.stride[1] + kd) * 2;
    v_together = (my_row * (unsigned)a.v.stride[1] + vd) * 2;
  }
  __device__ __forceinline__ int tiles() const { return WINDOW ? (span.count + CH - 1) / CH : tiles_of<KT>(a, count); }
  // The first key of each sixteen of tile t, one to a lane: asked for a tile before they are needed.
  __device__ __forceinline__ int look_up(int t) const {
    if constexpr (WINDOW) return span.first_key(t * CH + (int)(threadIdx.x % CH));
    return first_key(a, first, count, (long long)t * KT + 16 * (threadIdx.x % CH));
  }
  static __device__ __forceinline__ v4i spread(int of_lane) {
    static_assert(CH == 4, "tiles of 64 keys");
    return v4i{__builtin_amdgcn_readlane(of_lane, 0), __builtin_amdgcn_readlane(of_lane, 1), __builtin_amdgcn_readlane(of_lane, 2),
               __builtin_amdgcn_readlane(of_lane, 3)};
  }
  // The tile of these keys into one of the buffers.
  template <int BUFFER>
  __device__ __forceinline__ void load(v4i key0) const {
    constexpr unsigned buffer = BUFFER * KT * DP * 2;
    static_assert(KT == 64 && RP <= 32, "my_row * stride has 32 bits");
    // Most tiles: one behind the other, so that the addresses are a few additions.  The sixteens of a window ascend without a repetition, so that its
    // last one says it; those of lists of blocks of 16 come in any order.
    const bool follow = (key0[3] == key0[0] + 48) & (WINDOW || ((key0[1] == key0[0] + 16) & (key0[2] == key0[0] + 32)));
    if (near && follow && key0[0] <= a.keys - KT) {
      const elem *k = kp + key0[0] * a.k.stride[1], *v = vp + key0[0] * a.v.stride[1];
      const auto all = [&](auto which) {
        constexpr int p = decltype(which)::value;
        load_to_lds_behind<buffer + p * NW * 1024>(k + p * RP * a.k.stride[1], k_together, k_to);
      };
      const auto all_v = [&](auto which) {
        constexpr int p = decltype(which)::value;
        load_to_lds_behind<buffer + p * NW * 1024>(v + p * RP * a.v.stride[1], v_together, v_to);
      };
      static_assert(PASSES == 2 || PASSES == 4, "passes of a tile");
      if (kd < a.dim) {
        all(std::integral_constant<int, 0>());
        all(std::integral_constant<int, 1>());
        if constexpr (PASSES == 4) all(std::integral_constant<int, 2>()), all(std::integral_constant<int, 3>());
      }
      if (vd < a.dim) {
        all_v(std::integral_constant<int, 0>());
        all_v(std::integral_constant<int, 1>());
        if constexpr (PASSES == 4) all_v(std::integral_constant<int, 2>()), all_v(std::integral_constant<int, 3>());
      }
      return;
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int at = RP == 16 ? key0[p] : __builtin_amdgcn_readfirstlane(my_row < 16 ? key0[p * RP / 16] : key0[p * RP / 16 + (RP > 16)]);
      const int from = min(at, a.keys - 1), room = a.keys - 1 - from;
      const elem *k16 = kp + from * a.k.stride[1], *v16 = vp + from * a.v.stride[1];
      long long ko = k_off, vo = v_off;
      if (room < 15) ko = min(in16, room) * a.k.stride[1] + kd, vo = min(in16, room) * a.v.stride[1] + vd;
      if (kd < a.dim) load_to_lds(k16 + ko, k_to + buffer + p * NW * 1024);
      if (vd < a.dim) load_to_lds(v16 + vo, v_to + buffer + p * NW * 1024);
    }
  }
};

int read_block(const char *what, const lapis_hip_block_args *p, bool backward, BlockArgs *a);
// Sizes of lists are left to the caller: block_m and rows.
int read_window(const char *what, const lapis_hip_window_args *p, bool backward, BlockArgs *a);
// dQ over windows, by lists of block_m queries; rowsum(dO * O) times `scale` and the log-sums in units of ln 2 are left in delta and logs.
void launch_window_dq(const BlockArgs &a, bool bf16, bool few, float *delta, float *logs, hipStream_t st);
// Queries a list gets where a workgroup has `rows` rows, a row for each head of the group.
inline void cut_queries(BlockArgs *a, int rows) {
  a->block_m = std::max(1, rows / std::max(a->group, 1));
  a->rows = a->heads ? (int)ceil_div(a->queries, a->block_m) : 0;
}

// Windows: no more workgroups of 128 rows than compute units, so that a SIMD would have one wavefront.  Then two sides of a workgroup share its
// keys, by tiles in turn, and join through LDS.  One side and two, forward and dQ: 2048 queries, 16 heads, window 2048, dim 128: 66.7 and 48.2 us, 98.6 and
// 78.9; 1024 queries, 32 heads over 8, window 512: 27.1 and 24.0, 40.3 and 37.1; window 100 of 1024 queries, 16 heads: 19.3 and 16.6, 23.6 and 22.4.
inline bool few_workgroups(const BlockArgs &a) {
  return (int64_t)a.batch * a.kv_heads * a.rows * ceil_div((int64_t)a.block_m * a.group, 128) <= device_cu_count();
}

}  // namespace lapis
