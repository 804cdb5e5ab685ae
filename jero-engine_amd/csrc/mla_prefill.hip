// mla_prefill.hip -- latent attention over a paged cache: the expanded form, for prompts.
#include "mla.h"

namespace jero {

// Rows of the expanded keys and values: sequence s holds rows base(s) .. base(s) + min(lens[s],
// max_len) - 1, base the sum of the lengths before it; a sequence that ends past total has none.
__device__ __forceinline__ int mla_len(const LatentCache& c, int s) { return min(max(c.lens[s], 0), c.max_len); }

__device__ __forceinline__ bool mla_base(const LatentCache& c, int seq, int64_t total, int64_t& base) {
  base = 0;
  for (int s = 0; s < seq; s++) {
    const int n = mla_len(c, s);
    if (base + n <= total) base += n;
  }
  return base + mla_len(c, seq) <= total;
}

// kv[h][row][nope + v] = W[h] c, one workgroup per (position of a sequence, sequence).
template <typename KV>
__global__ void __launch_bounds__(256) mla_expand_kernel(LatentCache c, int nh, int wide,
                                                         const _Float16* __restrict__ w, int64_t total,
                                                         float* __restrict__ kv) {
  __shared__ float s_c[kMlaMaxRank];
  const int j = blockIdx.x, seq = blockIdx.y;
  int64_t base;
  if (j >= mla_len(c, seq) || !mla_base(c, seq, total, base)) return;
  const int64_t at = mla_row(c, seq, j);
  const KV* row = static_cast<const KV*>(c.rows) + at;
  for (int r = threadIdx.x; r < c.rank; r += 256) s_c[r] = at < 0 ? 0.f : float(row[r]);
  __syncthreads();
  for (int o = threadIdx.x; o < nh * wide; o += 256) {
    const _Float16* wr = w + int64_t(o) * c.rank;
    float s = 0.f;
    for (int r = 0; r < c.rank; r++) s += s_c[r] * float(wr[r]);
    kv[(int64_t(o / wide) * total + base + j) * wide + o % wide] = s;
  }
}

template <typename X, typename KV>
__global__ void __launch_bounds__(256) mla_prefill_kernel(LatentCache c, const X* __restrict__ q, int64_t q_stride,
                                                          int h0, int nope, int v_dim, const float* __restrict__ kv,
                                                          int64_t total, float scale, MlaRope rope, X* __restrict__ out,
                                                          int64_t out_stride) {
  __shared__ float s_q[256];
  __shared__ float s_o[4][256];
  __shared__ float s_m[4], s_l[4];
  const int t = blockIdx.x, h = h0 + blockIdx.y;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int wide = nope + v_dim, qw = nope + c.rope;
  int seq, pos;
  if (!mla_locate(c, t, lane, seq, pos)) return;
  int64_t base;
  const bool fits = mla_base(c, seq, total, base);
  const X* qr = q + t * q_stride + int64_t(h) * qw;
  for (int i = threadIdx.x; i < nope; i += 256) s_q[i] = float(qr[i]) * scale;
  if (int(threadIdx.x) < c.rope / 2) {
    const int i = threadIdx.x;
    const float a = float(qr[nope + 2 * i]), b = float(qr[nope + 2 * i + 1]);
    const float2 cs = rope.on ? mla_cos_sin(rope, i, pos) : make_float2(1.f, 0.f);
    s_q[nope + 2 * i] = (a * cs.x - b * cs.y) * scale;
    s_q[nope + 2 * i + 1] = (a * cs.y + b * cs.x) * scale;
  }
  __syncthreads();
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const int end = fits ? min(min(pos + 1, c.max_len), mla_len(c, seq)) : 0;
  for (int j = wv; j < end; j += 4) {
    const int64_t at = mla_row(c, seq, j);
    if (at < 0) continue;
    const KV* row = static_cast<const KV*>(c.rows) + at + c.rank;
    const float* kr = kv + (int64_t(blockIdx.y) * total + base + j) * wide;
    float s = 0.f;
    for (int i = lane; i < qw; i += 64) s += s_q[i] * (i < nope ? kr[i] : float(row[i - nope]));
    s = wave_sum_dpp(s);
    const float mn = fmaxf(m, s);
    const float a = mn == m ? 1.f : expf(m - mn), p = expf(s - mn);
    l = l * a + p;
    m = mn;
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = acc[i] * a + (lane + 64 * i < v_dim ? p * kr[nope + lane + 64 * i] : 0.f);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) s_o[wv][lane + 64 * i] = acc[i];
  if (lane == 0) s_m[wv] = m, s_l[wv] = l;
  __syncthreads();
  for (int v = threadIdx.x; v < v_dim; v += 256) {
    float M = -INFINITY;
    for (int w = 0; w < 4; w++) M = s_l[w] > 0.f ? fmaxf(M, s_m[w]) : M;
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; w++) {
      if (!(s_l[w] != 0.f)) continue;
      const float e = expf(s_m[w] - M);
      num += e * s_o[w][v];
      den += e * s_l[w];
    }
    out[t * out_stride + int64_t(h) * v_dim + v] = X(den != 0.f ? num / den : 0.f);
  }
}

}  // namespace jero

using namespace jero;

extern "C" size_t jero_hip_mla_prefill_workspace_bytes(const jero_latent_cache* cache, int act_dtype, int n_heads,
                                                       int nope_dim, int v_dim, int64_t total_len) {
  (void)act_dtype;
  if (!cache || n_heads < 1 || nope_dim < 1 || v_dim < 1 || total_len < 1) return 0;
  const size_t one = size_t(total_len) * (nope_dim + v_dim) * sizeof(float);
  const size_t most = one > (size_t(1) << 30) ? 1 : (size_t(1) << 30) / one;
  return one * (size_t(n_heads) < most ? size_t(n_heads) : most);
}

extern "C" int jero_hip_mla_prefill_attention(const jero_latent_cache* cache, int act_dtype, const void* q_dev,
                                              int64_t q_stride, int64_t n_tokens, int n_heads, int nope_dim, int v_dim,
                                              const void* kv_b_dev, int64_t total_len, float scale, float rope_theta,
                                              void* out_dev, int64_t out_stride, void* workspace_dev,
                                              size_t workspace_bytes, void* stream) {
  static const char* const kName = "mla_prefill_attention";
  int rc = mla_check_attention(cache, act_dtype, q_dev, q_stride, n_tokens, n_heads, nope_dim, v_dim, kv_b_dev,
                               kv_b_dev, scale, out_dev, out_stride, kName);
  if (rc) return rc;
  if (nope_dim + cache->rope_dim > 256)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, "mla_prefill_attention: nope_dim + rope_dim above 256");
  if (total_len < 1 || total_len > INT32_MAX)
    return fail(JERO_ERR_TENSOR_BOUNDS, "mla_prefill_attention: total_len must be 1 to 2^31 - 1");
  MlaRope rope;
  if ((rc = mla_rope_of(rope_theta, cache->rope_dim, &rope))) return rc;
  const size_t one = jero_hip_mla_prefill_workspace_bytes(cache, act_dtype, 1, nope_dim, v_dim, total_len);
  void* ws = workspace_dev;
  if (!ws) {
    workspace_bytes = jero_hip_mla_prefill_workspace_bytes(cache, act_dtype, n_heads, nope_dim, v_dim, total_len);
    if ((rc = workspace(workspace_bytes, &ws))) return rc;
  }
  if (workspace_bytes < one)
    return fail(JERO_ERR_TENSOR_BOUNDS, "mla_prefill_attention: workspace of " + std::to_string(workspace_bytes) +
                                            " bytes, need " + std::to_string(one));
  if (reinterpret_cast<uintptr_t>(ws) & 255u)
    return fail(JERO_ERR_INVALID_ARGUMENT, "mla_prefill_attention: workspace must be 256-byte aligned");
  const LatentCache c = mla_cache_of(cache, n_tokens);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int wide = nope_dim + v_dim;
  const int per = int(workspace_bytes / one < size_t(n_heads) ? workspace_bytes / one : size_t(n_heads));
  float* kv = static_cast<float*>(ws);
  for (int h0 = 0; h0 < n_heads; h0 += per) {
    const int nh = n_heads - h0 < per ? n_heads - h0 : per;
    const _Float16* w = static_cast<const _Float16*>(kv_b_dev) + int64_t(h0) * wide * c.rank;
    const dim3 ge{unsigned(c.max_len), unsigned(c.n_seqs), 1}, ga{unsigned(n_tokens), unsigned(nh), 1};
    if (cache->kv_dtype == JERO_KV_F16)
      hipLaunchKernelGGL((mla_expand_kernel<_Float16>), ge, dim3(256), 0, s, c, nh, wide, w, total_len, kv);
    else
      hipLaunchKernelGGL((mla_expand_kernel<float>), ge, dim3(256), 0, s, c, nh, wide, w, total_len, kv);
    if ((rc = check_launch("mla expand"))) return rc;
#define JERO_PREFILL(X, KV)                                                                                           \
  hipLaunchKernelGGL((mla_prefill_kernel<X, KV>), ga, dim3(256), 0, s, c, static_cast<const X*>(q_dev), q_stride, h0, \
                     nope_dim, v_dim, kv, total_len, scale, rope, static_cast<X*>(out_dev), out_stride)
    if (act_dtype == JERO_F16) JERO_PREFILL(_Float16, _Float16);
    else if (cache->kv_dtype == JERO_KV_F16) JERO_PREFILL(float, _Float16);
    else JERO_PREFILL(float, float);
#undef JERO_PREFILL
    if ((rc = check_launch("mla prefill"))) return rc;
  }
  return JERO_OK;
}
