// What the forward and backward kernels of block-sparse attention are given.
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

// Tiles of KT keys that a list has.  They are numbered with 31 bits: more would be 2^36 keys of one list, of the 2^30 there are.
template <int KT>
__device__ __forceinline__ int tiles_of(const BlockArgs &a, int count) {
  return a.keys > 0 ? (int)min((((long long)count << a.block_n_log2) + KT - 1) / KT, 0x7fffff00ll) : 0;
}

// Tiles of KT keys and values of a list on their way into two LDS buffers each, a workgroup of NW wavefronts sharing the
// work: sixteen rows at a time lie in one place.  A key that is not there is read from the last one: whoever uses the tile
// gives it no weight, and looks for values that are no numbers wherever a mask cuts.
template <typename T, int DP, int NW, int KT, bool V_BY_COLUMNS>
struct KeyTiles {
  typedef typename T::elem elem;
  static constexpr int PIECES = DP / 8, RP = NW * 64 / PIECES, PASSES = KT / RP, CH = KT / 16;
  static_assert(RP % 16 == 0, "a thread has the same row of each sixteen");
  const BlockArgs &a;
  const int first, count, wave, my_row, in16, kd, vd;
  const elem *kp, *vp;
  long long k_off, v_off;
  unsigned k_to, v_to;

  __device__ __forceinline__ KeyTiles(const BlockArgs &a_, int b, int kh, int first_, int count_, int tid, const elem *k_tile, const elem *v_tile)
      : a(a_), first(first_), count(count_), wave(__builtin_amdgcn_readfirstlane(tid >> 6)), my_row(tid / PIECES), in16(my_row & 15),
        kd(((tid % PIECES) ^ turn<DP>(my_row)) * 8), vd(((tid % PIECES) ^ (V_BY_COLUMNS ? column_turn<DP>(my_row) : turn<DP>(my_row))) * 8) {
    kp = (const elem *)a.k.data + b * a.k.stride[0] + kh * a.k.stride[2];
    vp = (const elem *)a.v.data + b * a.v.stride[0] + kh * a.v.stride[2];
    k_off = in16 * a.k.stride[1] + kd;
    v_off = in16 * a.v.stride[1] + vd;
    k_to = lds_address(k_tile) + wave * 1024;
    v_to = lds_address(v_tile) + wave * 1024;
  }
  __device__ __forceinline__ int tiles() const { return tiles_of<KT>(a, count); }
  // The first key of each sixteen of tile t, one to a lane: asked for a tile before they are needed.
  __device__ __forceinline__ int look_up(int t) const { return first_key(a, first, count, (long long)t * KT + 16 * (threadIdx.x % CH)); }
  static __device__ __forceinline__ v4i spread(int of_lane) {
    static_assert(CH == 4, "tiles of 64 keys");
    return v4i{__builtin_amdgcn_readlane(of_lane, 0), __builtin_amdgcn_readlane(of_lane, 1), __builtin_amdgcn_readlane(of_lane, 2),
               __builtin_amdgcn_readlane(of_lane, 3)};
  }
  // The tile of these keys into one of the buffers.
  template <int BUFFER>
  __device__ __forceinline__ void load(v4i key0) const {
    constexpr unsigned buffer = BUFFER * KT * DP * 2;
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

}  // namespace lapis
