// mla.hip -- latent attention over a paged cache: appending rows, and the absorbed form.
#include "mla.h"

#include <cmath>

namespace jero {

// ---------------------------------------------------------------- append

// One wave per token row: lane l holds elements 8l .. 8l + 7 of the latent, the first rope / 2 lanes a
// pair of the key part each.  The sum of squares is f32; the row is rounded once, to the cache's type.
template <typename X, typename KV>
__global__ void __launch_bounds__(256) mla_append_kernel(LatentCache c, const X* __restrict__ x, int64_t x_stride,
                                                         const float* __restrict__ norm, float eps, MlaRope rope) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= c.n_tokens) return;
  int seq, pos;
  if (!mla_locate(c, t, lane, seq, pos) || pos < 0 || pos >= c.max_len) return;
  const int64_t at = mla_row(c, seq, pos);
  if (at < 0) return;
  const X* xr = x + t * x_stride;
  KV* row = static_cast<KV*>(const_cast<void*>(c.rows)) + at;
  float v[8];
  float ss = 0.f;
  const bool in = 8 * lane < c.rank;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    v[e] = in ? float(xr[8 * lane + e]) : 0.f;
    ss += v[e] * v[e];
  }
  if (norm) {
    ss = wave_sum_dpp(ss);
    const float inv = 1.0f / sqrtf(ss / float(c.rank) + eps);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = in ? v[e] * inv * norm[8 * lane + e] : 0.f;
  }
  if (in)
#pragma unroll
    for (int e = 0; e < 8; e++) row[8 * lane + e] = KV(v[e]);
  if (lane < c.rope / 2) {
    const float a = float(xr[c.rank + 2 * lane]), b = float(xr[c.rank + 2 * lane + 1]);
    const float2 cs = rope.on ? mla_cos_sin(rope, lane, pos) : make_float2(1.f, 0.f);
    row[c.rank + 2 * lane] = KV(a * cs.x - b * cs.y);
    row[c.rank + 2 * lane + 1] = KV(a * cs.y + b * cs.x);
  }
}

// ---------------------------------------------------------------- absorbed attention

// q'[t][h] = [ q_n W_uk[h] | rotated q_p ] in f32, one workgroup per (token, head).
template <typename X>
__global__ void __launch_bounds__(256) mla_absorb_kernel(LatentCache c, const X* __restrict__ q, int64_t q_stride,
                                                         int nope, const _Float16* __restrict__ k_b, MlaRope rope,
                                                         float* __restrict__ qa) {
  const int t = blockIdx.x, h = blockIdx.y, nh = gridDim.y;
  int seq, pos;
  if (!mla_locate(c, t, threadIdx.x & 63, seq, pos)) return;
  const X* qr = q + t * q_stride + int64_t(h) * (nope + c.rope);
  float* o = qa + (int64_t(t) * nh + h) * c.width;
  for (int r = threadIdx.x; r < c.rank; r += 256) {
    const _Float16* w = k_b + (int64_t(h) * c.rank + r) * nope;
    float s = 0.f;
    for (int n = 0; n < nope; n++) s += float(qr[n]) * float(w[n]);
    o[r] = s;
  }
  if (int(threadIdx.x) < c.rope / 2) {
    const int i = threadIdx.x;
    const float a = float(qr[nope + 2 * i]), b = float(qr[nope + 2 * i + 1]);
    const float2 cs = rope.on ? mla_cos_sin(rope, i, pos) : make_float2(1.f, 0.f);
    o[c.rank + 2 * i] = a * cs.x - b * cs.y;
    o[c.rank + 2 * i + 1] = a * cs.y + b * cs.x;
  }
}

// The attended latent o[t][h][rank] in f32, one workgroup per (token, head), one pass: each wave takes
// every fourth position with a running maximum and sum, and the four merge at the end.
template <typename KV>
__global__ void __launch_bounds__(256) mla_attend_kernel(LatentCache c, const float* __restrict__ qa, float scale,
                                                         float* __restrict__ o) {
  constexpr int DL = (kMlaMaxRank + kMlaMaxRope) / kWave;
  constexpr int RL = kMlaMaxRank / kWave;
  __shared__ float s_o[4][kMlaMaxRank];
  __shared__ float s_m[4], s_l[4];
  const int t = blockIdx.x, h = blockIdx.y, nh = gridDim.y;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int seq, pos;
  if (!mla_locate(c, t, lane, seq, pos)) return;
  const float* qr = qa + (int64_t(t) * nh + h) * c.width;
  float q[DL], acc[RL];
#pragma unroll
  for (int i = 0; i < DL; i++) q[i] = lane + 64 * i < c.width ? qr[lane + 64 * i] * scale : 0.f;
#pragma unroll
  for (int i = 0; i < RL; i++) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const int end = min(pos + 1, c.max_len);
  for (int j = wv; j < end; j += 4) {
    const int64_t at = mla_row(c, seq, j);
    if (at < 0) continue;
    const KV* row = static_cast<const KV*>(c.rows) + at;
    float k[DL], s = 0.f;
#pragma unroll
    for (int i = 0; i < DL; i++) {
      k[i] = lane + 64 * i < c.width ? float(row[lane + 64 * i]) : 0.f;
      s += q[i] * k[i];
    }
    s = wave_sum_dpp(s);
    const float mn = fmaxf(m, s);
    const float a = mn == m ? 1.f : expf(m - mn), p = expf(s - mn);
    l = l * a + p;
    m = mn;
#pragma unroll
    for (int i = 0; i < RL; i++) acc[i] = acc[i] * a + p * k[i];
  }
#pragma unroll
  for (int i = 0; i < RL; i++) s_o[wv][lane + 64 * i] = acc[i];
  if (lane == 0) s_m[wv] = m, s_l[wv] = l;
  __syncthreads();
  for (int r = threadIdx.x; r < c.rank; r += 256) {
    float M = -INFINITY;
    for (int w = 0; w < 4; w++) M = s_l[w] > 0.f ? fmaxf(M, s_m[w]) : M;
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; w++) {
      if (!(s_l[w] != 0.f)) continue;  // no position of its own
      const float e = expf(s_m[w] - M);
      num += e * s_o[w][r];
      den += e * s_l[w];
    }
    o[(int64_t(t) * nh + h) * c.rank + r] = den != 0.f ? num / den : 0.f;
  }
}

// out[t][h][v] = o[t][h] . W_uv[h][v], one workgroup per (token, head).
template <typename X>
__global__ void __launch_bounds__(256) mla_values_kernel(LatentCache c, const float* __restrict__ o,
                                                         const _Float16* __restrict__ v_b, int v_dim,
                                                         X* __restrict__ out, int64_t out_stride) {
  const int t = blockIdx.x, h = blockIdx.y, nh = gridDim.y;
  int seq, pos;
  if (!mla_locate(c, t, threadIdx.x & 63, seq, pos)) return;
  const float* a = o + (int64_t(t) * nh + h) * c.rank;
  for (int v = threadIdx.x; v < v_dim; v += 256) {
    const _Float16* w = v_b + (int64_t(h) * v_dim + v) * c.rank;
    float s = 0.f;
    for (int r = 0; r < c.rank; r++) s += a[r] * float(w[r]);
    out[t * out_stride + int64_t(h) * v_dim + v] = X(s);
  }
}

// ---------------------------------------------------------------- checks

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int mla_check_cache(const jero_latent_cache* c, int64_t n_tokens, int act_dtype, const char* what) {
  const std::string w = std::string(what) + ": ";
  if (!c || !c->rows_dev || !c->table_dev || !c->lens_dev) return fail(JERO_ERR_INVALID_ARGUMENT, w + "null pointer");
  if (!aligned16(c->rows_dev)) return fail(JERO_ERR_INVALID_ARGUMENT, w + "the cache must be 16-byte aligned");
  if (!aligned4(c->table_dev) || !aligned4(c->lens_dev) || !aligned4(c->starts_dev))
    return fail(JERO_ERR_INVALID_ARGUMENT, w + "table, lens and starts must be 4-byte aligned");
  if (c->kv_dtype != JERO_KV_F32 && c->kv_dtype != JERO_KV_F16)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, w + "kv_dtype must be JERO_KV_F32 or JERO_KV_F16");
  if (act_dtype != JERO_F32 && act_dtype != JERO_F16)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, w + "activations must be JERO_F32 or JERO_F16");
  if (c->rank < 8 || c->rank % 8 || c->rank > kMlaMaxRank)
    return fail(JERO_ERR_CAPABILITY_MISMATCH,
                w + "rank " + std::to_string(c->rank) + " is not a multiple of 8 up to " + std::to_string(kMlaMaxRank));
  if (c->rope_dim < 8 || c->rope_dim % 8 || c->rope_dim > kMlaMaxRope)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, w + "rope_dim " + std::to_string(c->rope_dim) +
                                                  " is not a multiple of 8 up to " + std::to_string(kMlaMaxRope));
  if (c->block_size < 1 || c->block_size > (1 << 20) || (c->block_size & (c->block_size - 1)))
    return fail(JERO_ERR_CAPABILITY_MISMATCH,
                w + "block_size " + std::to_string(c->block_size) + " is not a power of two up to 2^20");
  if (n_tokens < 1 || c->n_seqs < 1 || c->n_blocks < 1 || c->max_len < 1)
    return fail(JERO_ERR_TENSOR_BOUNDS, w + "no tokens, sequences, blocks or positions");
  if (n_tokens > (1 << 22) || c->n_seqs > (1 << 22) || c->n_blocks > INT32_MAX)
    return fail(JERO_ERR_TENSOR_BOUNDS, w + "more than 2^22 tokens or sequences, or 2^31 blocks");
  if (!c->starts_dev && n_tokens != c->n_seqs)
    return fail(JERO_ERR_TENSOR_BOUNDS, w + std::to_string(n_tokens) + " tokens of " + std::to_string(c->n_seqs) +
                                            " sequences without their starts");
  if (c->max_len > JERO_MAX_LATENT_POSITIONS)
    return fail(JERO_ERR_CONTEXT_LENGTH_EXCEEDED,
                w + "more than " + std::to_string(JERO_MAX_LATENT_POSITIONS) + " positions");
  if (c->table_stride < 1 || c->table_stride > INT32_MAX || c->max_len > c->table_stride * c->block_size)
    return fail(JERO_ERR_TENSOR_BOUNDS, w + std::to_string(c->table_stride) + " blocks a sequence do not hold " +
                                            std::to_string(c->max_len) + " positions");
  return JERO_OK;
}

LatentCache mla_cache_of(const jero_latent_cache* c, int64_t n_tokens) {
  LatentCache k{};
  k.rows = c->rows_dev;
  k.table = c->table_dev;
  k.lens = c->lens_dev;
  k.starts = c->starts_dev;
  k.table_stride = c->table_stride;
  k.n_blocks = uint32_t(c->n_blocks);
  k.n_seqs = int(c->n_seqs);
  k.n_tokens = int(n_tokens);
  k.max_len = int(c->max_len);
  k.shift = __builtin_ctz(unsigned(c->block_size));
  k.rank = c->rank;
  k.rope = c->rope_dim;
  k.width = c->rank + c->rope_dim;
  return k;
}

int mla_rope_of(float theta, int rope_dim, MlaRope* out) {
  *out = MlaRope{};
  if (theta == 0.f) return JERO_OK;
  if (!(theta > 0.f) || !std::isfinite(theta))
    return fail(JERO_ERR_INVALID_ARGUMENT, "rope_theta must be positive, or 0 for rotated rows");
  out->on = 1;
  for (int i = 0; i < rope_dim / 2; i++)
    out->turns[i] = std::pow(double(theta), -2.0 * i / rope_dim) / 6.283185307179586476925;
  return JERO_OK;
}

int mla_check_attention(const jero_latent_cache* c, int act_dtype, const void* q, int64_t q_stride, int64_t n_tokens,
                        int n_heads, int nope, int v, const void* w0, const void* w1, float scale, const void* out,
                        int64_t out_stride, const char* what) {
  int rc = mla_check_cache(c, n_tokens, act_dtype, what);
  if (rc) return rc;
  const std::string w = std::string(what) + ": ";
  if (act_dtype == JERO_F16 && c->kv_dtype != JERO_KV_F16)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, w + "f16 activations need an f16 cache");
  if (!q || !w0 || !w1 || !out) return fail(JERO_ERR_INVALID_ARGUMENT, w + "null pointer");
  if (!aligned16(q) || !aligned16(w0) || !aligned16(w1) || !aligned16(out))
    return fail(JERO_ERR_INVALID_ARGUMENT, w + "q, weights and out must be 16-byte aligned");
  if (n_heads < 1) return fail(JERO_ERR_TENSOR_BOUNDS, w + "no heads");
  if (n_heads > 1024) return fail(JERO_ERR_CAPABILITY_MISMATCH, w + "more than 1024 heads");
  if (nope < 8 || nope % 8 || nope > 256 || v < 8 || v % 8 || v > 256)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, w + "nope_dim and v_dim must be multiples of 8 up to 256");
  if (q_stride < int64_t(n_heads) * (nope + c->rope_dim) || out_stride < int64_t(n_heads) * v)
    return fail(JERO_ERR_TENSOR_BOUNDS, w + "rows overlap: a stride is below its row's length");
  if (q_stride % 8 || out_stride % 8)
    return fail(JERO_ERR_INVALID_ARGUMENT, w + "strides must be multiples of 8 elements");
  if (!std::isfinite(scale)) return fail(JERO_ERR_INVALID_ARGUMENT, w + "scale must be finite");
  return JERO_OK;
}

static int absorbed_workspace(size_t need, void** ws, size_t have, const char* what) {
  if (!*ws) return workspace(need, ws);
  if (have < need)
    return fail(JERO_ERR_TENSOR_BOUNDS, std::string(what) + ": workspace of " + std::to_string(have) + " bytes, need " +
                                            std::to_string(need));
  if (reinterpret_cast<uintptr_t>(*ws) & 255u)
    return fail(JERO_ERR_INVALID_ARGUMENT, std::string(what) + ": workspace must be 256-byte aligned");
  return JERO_OK;
}

}  // namespace jero

using namespace jero;

extern "C" int jero_hip_mla_append(const jero_latent_cache* cache, int act_dtype, const void* x_dev, int64_t x_stride,
                                   int64_t n_tokens, const float* norm_dev, float eps, float rope_theta, void* stream) {
  int rc = mla_check_cache(cache, n_tokens, act_dtype, "mla_append");
  if (rc) return rc;
  if (!x_dev) return fail(JERO_ERR_INVALID_ARGUMENT, "mla_append: null pointer");
  if (reinterpret_cast<uintptr_t>(x_dev) & (act_dtype == JERO_F32 ? 3u : 1u) || !aligned4(norm_dev))
    return fail(JERO_ERR_INVALID_ARGUMENT, "mla_append: x and norm must be aligned to their elements");
  if (x_stride < cache->rank + cache->rope_dim)
    return fail(JERO_ERR_TENSOR_BOUNDS, "mla_append: rows overlap: the stride is below the row's length");
  if (norm_dev && !(eps >= 0.f && std::isfinite(eps)))
    return fail(JERO_ERR_INVALID_ARGUMENT, "mla_append: eps must be finite and not negative");
  MlaRope rope;
  if ((rc = mla_rope_of(rope_theta, cache->rope_dim, &rope))) return rc;
  const LatentCache c = mla_cache_of(cache, n_tokens);
  const dim3 grid(unsigned((n_tokens + 3) / 4));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = cache->kv_dtype == JERO_KV_F16;
#define JERO_APPEND(X, KV)                                                                                          \
  hipLaunchKernelGGL((mla_append_kernel<X, KV>), grid, dim3(256), 0, s, c, static_cast<const X*>(x_dev), x_stride, \
                     norm_dev, eps, rope)
  if (act_dtype == JERO_F32) {
    if (f16) JERO_APPEND(float, _Float16);
    else JERO_APPEND(float, float);
  } else {
    if (f16) JERO_APPEND(_Float16, _Float16);
    else JERO_APPEND(_Float16, float);
  }
#undef JERO_APPEND
  return check_launch("mla_append");
}

extern "C" size_t jero_hip_mla_absorbed_workspace_bytes(const jero_latent_cache* cache, int64_t n_tokens, int n_heads) {
  if (!cache || n_tokens < 1 || n_heads < 1) return 0;
  return size_t(n_tokens) * n_heads * (2 * size_t(cache->rank) + cache->rope_dim) * sizeof(float);
}

extern "C" int jero_hip_mla_absorbed_attention(const jero_latent_cache* cache, int act_dtype, const void* q_dev,
                                               int64_t q_stride, int64_t n_tokens, int n_heads, int nope_dim, int v_dim,
                                               const void* k_b_dev, const void* v_b_dev, float scale, float rope_theta,
                                               void* out_dev, int64_t out_stride, void* workspace_dev,
                                               size_t workspace_bytes, void* stream) {
  static const char* const kName = "mla_absorbed_attention";
  int rc = mla_check_attention(cache, act_dtype, q_dev, q_stride, n_tokens, n_heads, nope_dim, v_dim, k_b_dev, v_b_dev,
                               scale, out_dev, out_stride, kName);
  if (rc) return rc;
  MlaRope rope;
  if ((rc = mla_rope_of(rope_theta, cache->rope_dim, &rope))) return rc;
  void* ws = workspace_dev;
  if ((rc = absorbed_workspace(jero_hip_mla_absorbed_workspace_bytes(cache, n_tokens, n_heads), &ws, workspace_bytes,
                               kName)))
    return rc;
  const LatentCache c = mla_cache_of(cache, n_tokens);
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* qa = static_cast<float*>(ws);
  float* o = qa + n_tokens * n_heads * c.width;
  const dim3 grid{unsigned(n_tokens), unsigned(n_heads), 1};
  const _Float16 *kb = static_cast<const _Float16*>(k_b_dev), *vb = static_cast<const _Float16*>(v_b_dev);
  if (act_dtype == JERO_F32)
    hipLaunchKernelGGL((mla_absorb_kernel<float>), grid, dim3(256), 0, s, c, static_cast<const float*>(q_dev), q_stride,
                       nope_dim, kb, rope, qa);
  else
    hipLaunchKernelGGL((mla_absorb_kernel<_Float16>), grid, dim3(256), 0, s, c, static_cast<const _Float16*>(q_dev),
                       q_stride, nope_dim, kb, rope, qa);
  if ((rc = check_launch("mla absorb"))) return rc;
  if (cache->kv_dtype == JERO_KV_F16)
    hipLaunchKernelGGL((mla_attend_kernel<_Float16>), grid, dim3(256), 0, s, c, qa, scale, o);
  else
    hipLaunchKernelGGL((mla_attend_kernel<float>), grid, dim3(256), 0, s, c, qa, scale, o);
  if ((rc = check_launch("mla attend"))) return rc;
  if (act_dtype == JERO_F32)
    hipLaunchKernelGGL((mla_values_kernel<float>), grid, dim3(256), 0, s, c, o, vb, v_dim, static_cast<float*>(out_dev),
                       out_stride);
  else
    hipLaunchKernelGGL((mla_values_kernel<_Float16>), grid, dim3(256), 0, s, c, o, vb, v_dim,
                       static_cast<_Float16*>(out_dev), out_stride);
  return check_launch("mla values");
}
