// What the forward and backward kernels of block-sparse attention are given.
#pragma once
#include "attn.hpp"

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
__device__ __forceinline__ void entries_of(const BlockArgs &a, long long row, int *first, int *count) {
  const long long lo = min(max((long long)a.pos[row], 0ll), a.nnz), hi = min(max((long long)a.pos[row + 1], lo), a.nnz);
  *first = (int)lo;
  *count = (int)(hi - lo);
}

int read_block(const char *what, const lapis_hip_block_args *p, bool backward, BlockArgs *a);

}  // namespace lapis
