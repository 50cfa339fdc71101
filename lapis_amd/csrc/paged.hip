// Attention of one new token of each sequence over the pages of a cache that a CSR row lists.
#include "attn.hpp"

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
  int seqs, heads, kv_heads, dim, page_log2;
  bool each;  // a list per key-value head
  const int *pos, *crd, *tokens;
  float *lse;
  float scale;
};

// Pages that a row lists and tokens that count in them, whatever pos and tokens hold.
__device__ __forceinline__ void list_of(const PagedArgs &a, long long row, int *first, int *tokens) {
  const long long lo = min(max((long long)a.pos[row], 0ll), a.nnz), hi = min(max((long long)a.pos[row + 1], lo), a.nnz);
  *first = (int)lo;
  *tokens = (int)max(0ll, min((long long)a.tokens[row], (hi - lo) << a.page_log2));
}

// One wavefront per (sequence, head): 64 tokens at a time, a token per lane for the scores, then elements of the row
// per lane for the sum.
template <typename T, bool F8>
__global__ __launch_bounds__(64) void paged_simple_kernel(PagedArgs a) {
  typedef typename T::elem elem;
  const int lane = threadIdx.x, s = blockIdx.y, h = blockIdx.x, kh = h / (a.heads / a.kv_heads);
  __shared__ float q[kMaxDim], weight[64];
  __shared__ long long at[64];
  const elem *qp = (const elem *)a.q + s * a.q_stride[0] + h * a.q_stride[1];
  for (int d = lane; d < a.dim; d += 64) q[d] = (float)qp[d] * a.scale;
  int first, tokens;
  list_of(a, a.each ? (long long)s * a.kv_heads + kh : s, &first, &tokens);
  float m = -INFINITY, l = 0.f, acc[kMaxDim / 64] = {};
  __syncthreads();
  for (int t0 = 0; t0 < tokens; t0 += 64) {
    const int t = t0 + lane;
    float score = -INFINITY;
    long long from = -1;
    float vs = 1.f;
    if (t < tokens) {
      const int page = a.crd[first + (t >> a.page_log2)];
      if (page >= 0 && page < a.pages) {
        const int in = t & ((1 << a.page_log2) - 1);
        from = page * a.stride[0] + kh * a.stride[1] + in * a.stride[2];
        float dot = 0.f, ks = 1.f;
        if (F8) {
          const long long sc = page * a.scale_stride[0] + kh * a.scale_stride[1] + in * a.scale_stride[2];
          ks = a.k_scale[sc], vs = a.v_scale[sc];
        }
        for (int d = 0; d < a.dim; d += 8) {
          float f[8];
          if (F8) widen_f8(*(const v2i *)(a.k + from + d), f);
          else widen<T>(*(const vec8<T> *)((const elem *)a.k + from + d), f);
          for (int e = 0; e < 8; ++e) dot += q[d + e] * f[e];
        }
        score = dot * ks;
      }
    }
    float top = score;
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float m_new = fmaxf(m, top), keep = m == m_new ? 1.f : expf(m - m_new);
    const float p = score == -INFINITY ? 0.f : expf(score - m_new);
    l = l * keep + group_sum<64>(p);
    m = m_new;
    __syncthreads();
    weight[lane] = p * vs;
    at[lane] = from;
    __syncthreads();
    for (int i = 0; i < kMaxDim / 64; ++i) acc[i] *= keep;
    for (int j = 0; j < min(64, tokens - t0); ++j) {
      if (at[j] < 0) continue;
      for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = i * 64 + lane;
        if (d >= a.dim) continue;
        const float x = F8 ? __builtin_amdgcn_cvt_f32_fp8((int)(unsigned char)a.v[at[j] + d], 0) : (float)((const elem *)a.v)[at[j] + d];
        acc[i] += weight[j] * x;
      }
    }
  }
  elem *op = (elem *)a.out + s * a.out_stride[0] + h * a.out_stride[1];
  for (int i = 0; i < kMaxDim / 64; ++i)
    if (i * 64 + lane < a.dim) op[i * 64 + lane] = (elem)(l == 0.f ? 0.f : acc[i] / l);
  if (a.lse && lane == 0) a.lse[(long long)s * a.heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

int read_paged(const char *what, const lapis_hip_kv_cache *c, const lapis_hip_paged_args *p, PagedArgs *a) {
  const int rc = check_cache(what, c);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(p, "%s: null arguments", what);
  LAPIS_REQUIRE(p->seqs >= 0 && p->seqs <= 65535 * 16 && p->heads >= 0 && p->heads <= 65535 && p->heads % c->heads == 0,
                "%s: %lld sequences and %lld heads over a cache of %d", what, (long long)p->seqs, (long long)p->heads, c->heads);
  LAPIS_REQUIRE(p->lists == p->seqs || p->lists == p->seqs * c->heads, "%s: %lld lists of pages for %lld sequences", what,
                (long long)p->lists, (long long)p->seqs);
  LAPIS_REQUIRE(p->nnz >= 0 && p->nnz <= INT32_MAX && p->nnz * c->page <= INT32_MAX, "%s: %lld pages listed", what, (long long)p->nnz);
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
  return LAPIS_HIP_OK;
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_paged_attention_work(const lapis_hip_kv_cache *cache, const lapis_hip_paged_args *args, int64_t *bytes) {
  PagedArgs a;
  const int rc = read_paged("paged_attention", cache, args, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  LAPIS_REQUIRE(bytes, "paged_attention: null result");
  *bytes = 0;
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
  const bool f8 = cache->dtype == LAPIS_HIP_F8E4M3, bf16 = args->dtype == LAPIS_HIP_BF16;
  const auto kernel = bf16 ? (f8 ? paged_simple_kernel<Bf16, true> : paged_simple_kernel<Bf16, false>)
                           : (f8 ? paged_simple_kernel<F16, true> : paged_simple_kernel<F16, false>);
  LAPIS_REQUIRE(a.seqs <= 65535, "paged_attention: %d sequences", a.seqs);
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.heads, (unsigned)a.seqs), dim3(64), 0, as_stream(stream), a);
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}
