// Attention over the blocks that a CSR structure lists, forward.
#include "blockattn.hpp"

namespace lapis {
namespace {

// One wavefront per query and head: a key per lane for the scores, elements of the row per lane for the sum.
template <typename T>
__global__ __launch_bounds__(64) void block_simple_kernel(BlockArgs a) {
  typedef typename T::elem elem;
  const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, kh = h / a.group;
  __shared__ float q[kMaxBlockDim], weight[64];
  const elem *qp = (const elem *)a.q.data + b * a.q.stride[0] + i * a.q.stride[1] + h * a.q.stride[2];
  const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + kh * a.k.stride[2];
  const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + kh * a.v.stride[2];
  for (int d = lane; d < a.dim; d += 64) q[d] = (float)qp[d] * a.scale;
  int first, count;
  entries_of(a, ((long long)b * a.kv_heads + kh) * a.rows + i / a.block_m, &first, &count);
  float m = -INFINITY, l = 0.f, acc[kMaxBlockDim / 64] = {};
  __syncthreads();
  const int block_n = 1 << a.block_n_log2;
  for (int e = 0; e < count; ++e) {
    const int block = a.crd[first + e];
    if (block < 0 || block >= a.columns) continue;
    for (int n0 = 0; n0 < block_n; n0 += 64) {
      const int key = (block << a.block_n_log2) + n0 + lane;
      float score = -INFINITY;
      const bool live = n0 + lane < block_n && key < a.keys && (!a.causal || key <= i + a.shift);
      if (live) {
        score = 0.f;
        for (int d = 0; d < a.dim; d += 8) {
          float f[8];
          widen<T>(*(const vec8<T> *)(kp + key * a.k.stride[1] + d), f);
          for (int x = 0; x < 8; ++x) score += q[d + x] * f[x];
        }
      }
      float top = score;
      for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
      const float m_new = fmaxf(m, top), keep = m == m_new ? 1.f : expf(m - m_new);
      const float p = !live || score == -INFINITY ? 0.f : expf(score - m_new);
      l = l * keep + group_sum<64>(p);
      m = m_new;
      __syncthreads();
      weight[lane] = p;
      const unsigned long long use = __ballot(live);
      __syncthreads();
      for (int x = 0; x < kMaxBlockDim / 64; ++x) acc[x] *= keep;
      for (int j = 0; j < 64; ++j) {
        if (!(use >> j & 1)) continue;
        for (int x = 0; x < kMaxBlockDim / 64; ++x)
          if (x * 64 + lane < a.dim) acc[x] += weight[j] * (float)vp[(key - lane + j) * a.v.stride[1] + x * 64 + lane];
      }
    }
  }
  elem *op = (elem *)a.out.data + b * a.out.stride[0] + i * a.out.stride[1] + h * a.out.stride[2];
  for (int x = 0; x < kMaxBlockDim / 64; ++x)
    if (x * 64 + lane < a.dim) op[x * 64 + lane] = (elem)(l == 0.f ? 0.f : acc[x] / l);
  if (a.lse && lane == 0) a.lse[((long long)b * a.heads + h) * a.queries + i] = l == 0.f ? -INFINITY : m + logf(l);
}

int read_view(const char *what, const lapis_hip_rows &r, View *v) {
  LAPIS_REQUIRE(r.data && aligned16(r.data) && strides_of_8(r.stride, 3),
                "%s: an operand that is null, not on a 16-byte boundary or with strides that are no multiples of 8", what);
  v->data = static_cast<char *>(r.data);
  for (int i = 0; i < 3; ++i) v->stride[i] = r.stride[i];
  return LAPIS_HIP_OK;
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
  a->block_m = (int)p->block_m;
  a->block_n_log2 = __builtin_ctz((unsigned)p->block_n);
  a->rows = (int)ceil_div(p->queries, p->block_m);
  a->columns = (int)ceil_div(p->keys, p->block_n);
  a->causal = p->causal != 0;
  a->shift = (int)(p->keys - p->queries);
  a->scale = p->scale;
  a->pos = p->pos;
  a->crd = p->crd;
  a->nnz = p->nnz;
  a->lse = p->lse;
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

}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_block_attention(const lapis_hip_block_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_block("block_attention", args, false, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0 || a.queries == 0 || a.heads == 0) return LAPIS_HIP_OK;
  const auto kernel = args->dtype == LAPIS_HIP_BF16 ? block_simple_kernel<Bf16> : block_simple_kernel<F16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.queries, (unsigned)a.heads, (unsigned)a.batch), dim3(64), 0, as_stream(stream), a);
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}
