// Attention over the blocks that a CSR structure lists, backward.
#include "blockattn.hpp"

namespace lapis {
namespace {

// rowsum(dout * out) of every (batch entry, head, query)
template <typename T>
__global__ __launch_bounds__(64) void delta_simple_kernel(BlockArgs a, float *delta) {
  typedef typename T::elem elem;
  const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const elem *x = (const elem *)a.dout.data + b * a.dout.stride[0] + i * a.dout.stride[1] + h * a.dout.stride[2];
  const elem *y = (const elem *)a.out.data + b * a.out.stride[0] + i * a.out.stride[1] + h * a.out.stride[2];
  float s = 0.f;
  for (int d = lane; d < a.dim; d += 64) s += (float)x[d] * (float)y[d];
  s = group_sum<64>(s);
  if (lane == 0) delta[((long long)b * a.heads + h) * a.queries + i] = s;
}

// P and dS of one query and one key
template <typename T>
__device__ __forceinline__ void pair_of(const BlockArgs &a, const float *q, const float *dout, const typename T::elem *k,
                                        const typename T::elem *v, float lse, float delta, float *p, float *ds) {
  float s = 0.f, dp = 0.f;
  for (int d = 0; d < a.dim; d += 8) {
    float f[8], g[8];
    widen<T>(*(const vec8<T> *)(k + d), f);
    widen<T>(*(const vec8<T> *)(v + d), g);
    for (int x = 0; x < 8; ++x) s += q[d + x] * f[x], dp += dout[d + x] * g[x];
  }
  *p = lse == -INFINITY ? 0.f : expf(s * a.scale - lse);
  *ds = *p * (dp - delta) * a.scale;
}

template <typename T>
__global__ __launch_bounds__(64) void dq_simple_kernel(BlockArgs a, const float *delta) {
  typedef typename T::elem elem;
  const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, kh = h / a.group;
  __shared__ float q[kMaxBlockDim], dout[kMaxBlockDim], weight[64];
  const elem *qp = (const elem *)a.q.data + b * a.q.stride[0] + i * a.q.stride[1] + h * a.q.stride[2];
  const elem *dp = (const elem *)a.dout.data + b * a.dout.stride[0] + i * a.dout.stride[1] + h * a.dout.stride[2];
  const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + kh * a.k.stride[2];
  const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + kh * a.v.stride[2];
  for (int d = lane; d < a.dim; d += 64) q[d] = (float)qp[d], dout[d] = (float)dp[d];
  const long long at = ((long long)b * a.heads + h) * a.queries + i;
  const float lse = a.lse[at], del = delta[at];
  int first, count;
  entries_of(a, ((long long)b * a.kv_heads + kh) * a.rows + i / a.block_m, &first, &count);
  float acc[kMaxBlockDim / 64] = {};
  const int block_n = 1 << a.block_n_log2;
  __syncthreads();
  for (int e = 0; e < count; ++e) {
    const int block = a.crd[first + e];
    if (block < 0 || block >= a.columns) continue;
    for (int n0 = 0; n0 < block_n; n0 += 64) {
      const int key = (block << a.block_n_log2) + n0 + lane;
      float p = 0.f, ds = 0.f;
      const bool live = n0 + lane < block_n && key < a.keys && (!a.causal || key <= i + a.shift);
      if (live) pair_of<T>(a, q, dout, kp + key * a.k.stride[1], vp + key * a.v.stride[1], lse, del, &p, &ds);
      __syncthreads();
      weight[lane] = ds;
      const unsigned long long use = __ballot(live);
      __syncthreads();
      for (int j = 0; j < 64; ++j) {
        if (!(use >> j & 1)) continue;
        for (int x = 0; x < kMaxBlockDim / 64; ++x)
          if (x * 64 + lane < a.dim) acc[x] += weight[j] * (float)kp[(key - lane + j) * a.k.stride[1] + x * 64 + lane];
      }
    }
  }
  elem *op = (elem *)a.dq.data + b * a.dq.stride[0] + i * a.dq.stride[1] + h * a.dq.stride[2];
  for (int x = 0; x < kMaxBlockDim / 64; ++x)
    if (x * 64 + lane < a.dim) op[x * 64 + lane] = (elem)acc[x];
}

// One wavefront per key: a query per lane, over the rows that list the key's block.
template <typename T>
__global__ __launch_bounds__(64) void dkv_simple_kernel(BlockArgs a, const float *delta) {
  typedef typename T::elem elem;
  const int lane = threadIdx.x, key = blockIdx.x, kh = blockIdx.y, b = blockIdx.z;
  __shared__ float k[kMaxBlockDim], v[kMaxBlockDim], wp[64], wds[64];
  const elem *kp = (const elem *)a.k.data + b * a.k.stride[0] + key * a.k.stride[1] + kh * a.k.stride[2];
  const elem *vp = (const elem *)a.v.data + b * a.v.stride[0] + key * a.v.stride[1] + kh * a.v.stride[2];
  for (int d = lane; d < a.dim; d += 64) k[d] = (float)kp[d], v[d] = (float)vp[d];
  float ak[kMaxBlockDim / 64] = {}, av[kMaxBlockDim / 64] = {};
  __syncthreads();
  for (int r = 0; r < a.rows; ++r) {
    int first, count, times = 0;
    entries_of(a, ((long long)b * a.kv_heads + kh) * a.rows + r, &first, &count);
    for (int e = lane; e < count; e += 64) times += a.crd[first + e] == key >> a.block_n_log2;
    times = group_sum<64>(times);
    if (times == 0) continue;
    const int q0 = r * a.block_m, n = min(a.block_m, a.queries - q0) * a.group;
    for (int x0 = 0; x0 < n; x0 += 64) {
      const int x = x0 + lane, i = q0 + x / a.group, h = kh * a.group + x % a.group;
      float p = 0.f, ds = 0.f;
      const bool live = x < n && (!a.causal || key <= i + a.shift);
      const elem *qp = nullptr, *dp = nullptr;
      if (live) {
        qp = (const elem *)a.q.data + b * a.q.stride[0] + i * a.q.stride[1] + h * a.q.stride[2];
        dp = (const elem *)a.dout.data + b * a.dout.stride[0] + i * a.dout.stride[1] + h * a.dout.stride[2];
        const long long at = ((long long)b * a.heads + h) * a.queries + i;
        pair_of<T>(a, k, v, qp, dp, a.lse[at], delta[at], &p, &ds);
      }
      const unsigned long long use = __ballot(live);
      __syncthreads();
      wp[lane] = p * times, wds[lane] = ds * times;
      __syncthreads();
      for (int j = 0; j < 64; ++j) {
        if (!(use >> j & 1)) continue;
        const int jx = x0 + j, ji = q0 + jx / a.group, jh = kh * a.group + jx % a.group;
        const elem *jq = (const elem *)a.q.data + b * a.q.stride[0] + ji * a.q.stride[1] + jh * a.q.stride[2];
        const elem *jd = (const elem *)a.dout.data + b * a.dout.stride[0] + ji * a.dout.stride[1] + jh * a.dout.stride[2];
        for (int y = 0; y < kMaxBlockDim / 64; ++y) {
          const int d = y * 64 + lane;
          if (d < a.dim) ak[y] += wds[j] * (float)jq[d], av[y] += wp[j] * (float)jd[d];
        }
      }
    }
  }
  elem *ok = (elem *)a.dk.data + b * a.dk.stride[0] + key * a.dk.stride[1] + kh * a.dk.stride[2];
  elem *ov = (elem *)a.dv.data + b * a.dv.stride[0] + key * a.dv.stride[1] + kh * a.dv.stride[2];
  for (int y = 0; y < kMaxBlockDim / 64; ++y)
    if (y * 64 + lane < a.dim) ok[y * 64 + lane] = (elem)ak[y], ov[y * 64 + lane] = (elem)av[y];
}

template <typename T>
void launch_backward(const BlockArgs &a, float *delta, hipStream_t st) {
  if (a.queries && a.heads) {
    const dim3 grid((unsigned)a.queries, (unsigned)a.heads, (unsigned)a.batch);
    hipLaunchKernelGGL(delta_simple_kernel<T>, grid, dim3(64), 0, st, a, delta);
    hipLaunchKernelGGL(dq_simple_kernel<T>, grid, dim3(64), 0, st, a, delta);
  }
  if (a.keys && a.kv_heads)
    hipLaunchKernelGGL(dkv_simple_kernel<T>, dim3((unsigned)a.keys, (unsigned)a.kv_heads, (unsigned)a.batch), dim3(64), 0, st, a, delta);
}

}  // namespace
}  // namespace lapis

using namespace lapis;

extern "C" int lapis_hip_block_attention_backward_work(const lapis_hip_block_args *args, int64_t *bytes) {
  LAPIS_REQUIRE(args && bytes, "block_attention_backward: null arguments");
  LAPIS_REQUIRE(args->batch >= 0 && args->heads >= 0 && args->queries >= 0, "block_attention_backward: a negative size");
  *bytes = 4 * args->batch * args->heads * args->queries;
  return LAPIS_HIP_OK;
}

extern "C" int lapis_hip_block_attention_backward(const lapis_hip_block_args *args, lapis_hip_stream_t stream) {
  LAPIS_CHECK_INIT();
  BlockArgs a;
  const int rc = read_block("block_attention_backward", args, true, &a);
  if (rc != LAPIS_HIP_OK) return rc;
  if (a.batch == 0) return LAPIS_HIP_OK;
  LAPIS_REQUIRE(args->work || a.queries == 0 || a.heads == 0, "block_attention_backward: null work");
  float *delta = static_cast<float *>(args->work);
  args->dtype == LAPIS_HIP_BF16 ? launch_backward<Bf16>(a, delta, as_stream(stream)) : launch_backward<F16>(a, delta, as_stream(stream));
  LAPIS_LAUNCH_CHECK();
  return LAPIS_HIP_OK;
}
