// paged_attention.hip -- attention over a paged key/value cache whose sequences may share their first positions:
// how a call is cut, the joining of its parts, and the entry point.
#include <algorithm>
#include <cmath>

#include "paged_attend.h"
#include "runtime.h"

namespace jero {

// Joins a row's (a token's head's) parts: the chunks of the shared positions, then those of its own.  DL lanes a part, four
// results each, PL parts of a row at a time.
template <typename X, int DL, int PL>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedCall c, PagedPlan p, X* __restrict__ out,
                                                          const float* __restrict__ part_o,
                                                          const float2* __restrict__ part_ml) {
  constexpr int R = 256 / (DL * PL);
  __shared__ f4_t s_v[R][PL][DL];
  __shared__ float s_l[R][PL];
  const int tid = threadIdx.x, d = 4 * (tid % DL), k0 = tid / DL % PL, r = tid / (DL * PL);
  const int64_t row = int64_t(blockIdx.x) * R + r;
  const int t = int(row / c.heads), h = int(row % c.heads);
  __shared__ int32_t s_starts[kSearchSeqs + 1];
  const int32_t* const starts = paged_starts(c, s_starts, tid);
  const int seen = t < c.n_tokens ? paged_visible(c, starts, t) : -1;
  const int shared = min(seen, c.shared_len);
  const int pre = p.pre_chunks && seen > 0 ? (shared + p.pre_len - 1) / p.pre_len : 0;
  const int own = seen > p.own_lo ? (seen - p.own_lo + p.own_len - 1) / p.own_len : 0;
  const int64_t step = int64_t(c.n_tokens) * c.heads;
  auto at = [&](int k) { return row + step * (k < pre ? k : p.pre_chunks + k - pre); };
  float m = -INFINITY;
  for (int k = tid % DL; k < pre + own; k += DL) m = fmaxf(m, part_ml[at(k)].x);
#pragma unroll
  for (int off = 1; off < DL; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f4_t v = {0.f, 0.f, 0.f, 0.f};
  // (eight parts' loads at a time)
  const int parts = pre + own;
  for (int k1 = k0; k1 < parts; k1 += 8 * PL) {
    float2 ml[8];
    f4_t o[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int k = k1 + i * PL;
      ml[i] = make_float2(-INFINITY, 0.f);
      o[i] = f4_t{0.f, 0.f, 0.f, 0.f};
      if (k < parts) {
        ml[i] = part_ml[at(k)];
        if (d < c.dim) o[i] = *reinterpret_cast<const f4_t*>(part_o + at(k) * c.dim + d);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float e = __builtin_amdgcn_exp2f(ml[i].x - ref);
      l += e * ml[i].y;
      v += e * o[i];
    }
  }
  if constexpr (PL > 1) {
    s_v[r][k0][tid % DL] = v;
    if (tid % DL == 0) s_l[r][k0] = l;
    __syncthreads();
  }
  if (k0 || d >= c.dim || seen < 0) return;
#pragma unroll
  for (int k = 1; k < PL; k++) v += s_v[r][k][tid % DL], l += s_l[r][k];
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  X* dst = out + t * c.out_stride + int64_t(h) * c.dim + d;
#pragma unroll
  for (int e = 0; e < 4; e++) dst[e] = X(v[e] * inv);
}

template <typename X>
static void launch_merge(const PagedCall& c, const PagedPlan& p, void* out, const float* part_o, const float2* part_ml,
                         hipStream_t s) {
  const int64_t rows = int64_t(c.n_tokens) * c.heads;
#define JERO_MERGE(DL, PL)                                                                                            \
  hipLaunchKernelGGL((paged_merge_kernel<X, DL, PL>), dim3(unsigned((rows * DL * PL + 255) / 256)), dim3(256), 0, s, c, p, \
                     static_cast<X*>(out), part_o, part_ml)
  // a row's lanes read eight parts at a time: more of them only where there are more parts (5 parts of 16384 rows of 128: 34 us
  // by eight, 11 by one)
  const int by = p.parts <= 8 ? 1 : p.parts <= 32 ? 2 : 8;
  if (c.dim <= 64) {
    if (by == 1) JERO_MERGE(16, 1);
    else if (by == 2) JERO_MERGE(16, 2);
    else JERO_MERGE(16, 8);
  } else if (c.dim <= 128) {
    if (by == 1) JERO_MERGE(32, 1);
    else if (by == 2) JERO_MERGE(32, 2);
    else JERO_MERGE(32, 8);
  } else {
    if (by == 1) JERO_MERGE(64, 1);
    else if (by == 2) JERO_MERGE(64, 2);
    else JERO_MERGE(64, 4);
  }
#undef JERO_MERGE
}

static int head_width(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

static PagedPlan paged_plan(const jero_paged_cache* k, bool f16, int64_t n_tokens, int n_heads) {
  PagedPlan p{};
  const int group = n_heads / k->n_heads_kv, hd = head_width(k->head_dim), kv = k->n_heads_kv;
  const int64_t shared = std::min<int64_t>(k->shared_blocks * k->block_size, k->max_len);
  const int64_t rows = n_tokens * group, each = (n_tokens + k->n_seqs - 1) / k->n_seqs * group;
  p.wide_rows = hd <= 128 && k->kv_dtype == JERO_KV_F16 ? 128 : 64;
  // Rows of all sequences go over the shared positions together where sequences do not fill tiles themselves and more than
  // 48 MB (24 of f32, whose rows cost more than their bytes) are spared.  Single tokens of 8, 32 and 128 sequences, 50 to 300
  // positions of their own, 8 heads of 128, f16, us apart and not: at 24 MB 15 and 14, 16 and 16, (33 MB) 29 and 25; at 48
  // MB 15 and 16, 16 and 18, (67) 30 and 28; at 160 MB 18 and 25, 18 and 26, 31 and 33.  Heads of 64 are even later, at 50 to
  // 160 MB.  An f32 cache: 25 and 20 (26 MB), 25 and 28 (33 MB), 55 and 53 (67 MB); at 160 MB 27 and 38, 28 and 40, (133) 57
  // and 62; of 45 calls drawn over all sizes the time not apart is 0.95 of that apart on average below 24 MB (0.59 to 1.21), 1.02
  // from 24 to 48 (0.69 to 1.23), 1.21 above (0.97 to 1.67).  128 x 4096 shared positions: 69 and 192.  Not where the two
  // parts of all rows would take more than 4 GiB.
  const double pair = 2.0 * kv * k->head_dim * (k->kv_dtype == JERO_KV_F16 ? 2 : 4);  // bytes of a position
  const double spared = double(k->n_seqs - 1) * shared * pair;
  const bool apart = k->n_seqs > 1 && each < p.wide_rows && spared >= (k->kv_dtype == JERO_KV_F16 ? 48e6 : 24e6) &&
                     n_tokens * n_heads * k->head_dim <= (int64_t(1) << 29);
  // Rows a sequence from which its own positions go by wide tiles, not by 16 rows at a time: 16 sequences of up to 2000, 8 heads
  // of 128, 32, 48, 64 and 96 rows each: f16 36, 41, 43 and 44 us wide, 37, 41, 46 and 65 by 16; f32 over f16 48, 56, 61 and
  // 64, and 39, 42, 48 and 66; f32 68, 68, 85 and 85, and 74, 91, 98 and 132.  Heads of 256, whose narrow tiles are one a CU,
  // 24 and 48 rows: f32 over f16 43 and 50 wide, 49 and 59 by 16; heads of 64, 48 and 80: 28 and 31, and 16 and 22.
  // Where wide tiles alone are two workgroups a CU they are taken from 17 rows on (74 sequences, 8 heads of 80, 24, 40 and 80
  // rows over 128 positions behind 736 shared: f32 over f16 43, 60 and 83 us wide, 49, 71 and 123 by 16).  74 sequences of 50
  // to 700, 8 heads, 20, 32 and 48 rows, wide and by 16: heads of 64 f16 31, 35, 36 and 29, 32, 49, f32 over f32 41, 45, 45
  // and 40, 47, 72; of 128 f16 44, 45, 47 and 42, 48, 77, f32 70, 75, 73 and 91, 102, 161; of 256 f16 79, 80, 88 and 96, 112,
  // 194.  f32 over f16 would want narrow tiles up to 32 rows there: heads of 64 40, 45, 45 and 26, 27, 41, of 128 67, 64, 63
  // and 45, 49, 77 (200 sequences 124, 128, 123 and 115, 124, 200); only heads of 256 have 100, 95, 88 and 116, 128, 209.
  const bool many = k->n_seqs * kv >= 512;
  p.own_wide = each > (many || hd == 256 ? kNarrowRows : hd == 64 ? 80 : f16 ? 48 : k->kv_dtype == JERO_KV_F16 ? 95 : 31);
  p.own_lo = apart ? int(shared) : 0;
  const int own_rows = p.own_wide ? p.wide_rows : kNarrowRows;
  const int64_t tiles = k->starts_dev ? rows / own_rows + k->n_seqs : n_tokens * ((group + own_rows - 1) / own_rows);
  p.own_tiles = int(tiles);
  const int64_t span = std::max<int64_t>(k->max_len - p.own_lo, 1);
  // Own positions in chunks where 512 workgroups, two a CU, would not come out otherwise (64 sequences of up to 1500, 8 heads:
  // one chunk 69 us, two 73; 32 of up to 800: one 20, four 27; one of 131072: 64 chunks 110, 128 119), of 256 and more.
  auto chunks = [&](int64_t blocks, int64_t span, int64_t want, int64_t least) {
    return std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, (span + least - 1) / least));
  };
  auto length = [](int64_t span, int64_t n) { return int(((span + n - 1) / n + 127) / 128 * 128); };
  p.own_len = length(span, chunks(tiles * kv, span, 512, 256));
  p.own_chunks = int((span + p.own_len - 1) / p.own_len);
  p.own_blocks = int(tiles * kv * p.own_chunks);
  if (apart) {
    // (8192 shared positions, 32, 64 and 128 rows: f16 31, 24 and 32 us wide, 21, 31 and 43 by 16)
    p.pre_wide = rows > 32;
    const int pre_rows = p.pre_wide ? p.wide_rows : kNarrowRows;
    p.pre_tiles = int((rows + pre_rows - 1) / pre_rows);
    // Chunks that take no longer than the call: with the cards' rates of a workgroup over the shared positions (us a position)
    // and of memory, four fifths of both phases' times one after the other.  64 f32 sequences, 8192 shared positions,
    // up to 1500 own: chunks of 1024 positions 67 us, of 512 73, of 256 79; 256 f16 sequences, 32768 and 700: chunks of
    // 8192 372 us, of 16384 430, of 4096 383; 7 sequences, 2048 (f32 cache): of 128 21, of 256 25.
    const double rate = p.pre_wide ? (f16 ? 0.04 : 0.06) * (hd / 128.0) : 0.01, memory = 5e6;
    const double both = double(p.pre_tiles) * kv * shared * rate / 512 + double(k->n_seqs) * span * 0.6 * pair / memory;
    const int64_t least = int64_t(std::max(128.0, 0.8 * both / rate));
    p.pre_len = length(shared, std::max<int64_t>(1, (shared + least - 1) / least));
    p.pre_chunks = int((shared + p.pre_len - 1) / p.pre_len);
    p.pre_blocks = p.pre_tiles * kv * p.pre_chunks;
  }
  p.parts = p.pre_chunks + p.own_chunks;
  return p;
}

static size_t part_bytes(const PagedPlan& p, int64_t n_tokens, int n_heads, int dim, size_t* ml) {
  if (p.parts == 1) return 0;
  const size_t rows = size_t(p.parts) * n_tokens * n_heads, o = (rows * dim * 4 + 255) & ~size_t(255);
  if (ml) *ml = o;
  return o + rows * 8;
}

static int check_paged(const jero_paged_cache* c, int64_t n_tokens, int n_heads) {
  auto bad = [](int status, const std::string& what) { return fail(status, "paged_attention: " + what); };
  auto aligned = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!c || !c->k_dev || !c->v_dev || !c->table_dev || !c->lens_dev) return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned(c->k_dev, 16) || !aligned(c->v_dev, 16))
    return bad(JERO_ERR_INVALID_ARGUMENT, "the cache must be 16-byte aligned");
  if (!aligned(c->table_dev, 4) || !aligned(c->lens_dev, 4) || !aligned(c->starts_dev, 4) || !aligned(c->shared_dev, 4))
    return bad(JERO_ERR_INVALID_ARGUMENT, "table, lens, starts and shared must be 4-byte aligned");
  if (c->kv_dtype != JERO_KV_F32 && c->kv_dtype != JERO_KV_F16)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "kv_dtype must be JERO_KV_F32 or JERO_KV_F16");
  if (c->head_dim < 8 || c->head_dim % 8 || c->head_dim > 256)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "head_dim " + std::to_string(c->head_dim) + " is not a multiple of 8 up to 256");
  if (c->block_size < 1 || c->block_size > (1 << 20) || (c->block_size & (c->block_size - 1)))
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "block_size " + std::to_string(c->block_size) + " is not a power of two up to 2^20");
  if (n_tokens < 1 || c->n_seqs < 1 || c->n_blocks < 1 || c->max_len < 1 || n_heads < 1 || c->n_heads_kv < 1)
    return bad(JERO_ERR_TENSOR_BOUNDS, "no tokens, sequences, blocks, positions or heads");
  if (n_heads > 1024) return bad(JERO_ERR_CAPABILITY_MISMATCH, "more than 1024 heads");
  if (n_heads % c->n_heads_kv) return bad(JERO_ERR_TENSOR_BOUNDS, "n_heads is not a multiple of n_heads_kv");
  if (n_tokens > (1 << 19) || c->n_seqs > (1 << 19) || c->n_blocks > INT32_MAX)
    return bad(JERO_ERR_TENSOR_BOUNDS, "more than 2^19 tokens or sequences, or 2^31 - 1 blocks");
  if (!c->starts_dev && n_tokens != c->n_seqs)
    return bad(JERO_ERR_TENSOR_BOUNDS, std::to_string(n_tokens) + " tokens of " + std::to_string(c->n_seqs) +
                                           " sequences without their starts");
  if (c->max_len > JERO_MAX_PAGED_POSITIONS)
    return bad(JERO_ERR_CONTEXT_LENGTH_EXCEEDED, "more than " + std::to_string(JERO_MAX_PAGED_POSITIONS) + " positions");
  if (c->table_stride < 1 || c->table_stride > INT32_MAX || c->max_len > c->table_stride * c->block_size)
    return bad(JERO_ERR_TENSOR_BOUNDS, std::to_string(c->table_stride) + " blocks a sequence do not hold " +
                                           std::to_string(c->max_len) + " positions");
  if (c->shared_blocks < 0 || (c->shared_blocks > 0 && !c->shared_dev) || c->shared_blocks > c->table_stride)
    return bad(JERO_ERR_TENSOR_BOUNDS, "shared_blocks without their ids, or more than a table row");
  if (n_tokens * n_heads > (1 << 25)) return bad(JERO_ERR_CAPABILITY_MISMATCH, "more than 2^25 rows of heads");
  if (c->n_seqs * c->n_heads_kv > (1 << 22))  // (each a workgroup, if only to see that it has no rows)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "more than 2^22 sequences times key heads");
  return JERO_OK;
}

}  // namespace jero

using namespace jero;

extern "C" size_t jero_hip_paged_attention_workspace_bytes(const jero_paged_cache* cache, int act_dtype, int64_t n_tokens,
                                                           int n_heads) {
  if (check_paged(cache, n_tokens, n_heads)) return 0;
  return part_bytes(paged_plan(cache, act_dtype == JERO_F16, n_tokens, n_heads), n_tokens, n_heads, cache->head_dim, nullptr);
}

extern "C" int jero_hip_paged_attention(const jero_paged_cache* cache, int act_dtype, const void* q_dev, int64_t q_stride,
                                        int64_t n_tokens, int n_heads, float scale, void* out_dev, int64_t out_stride,
                                        void* workspace_dev, size_t workspace_bytes, void* stream) {
  auto bad = [](int status, const char* what) { return fail(status, std::string("paged_attention: ") + what); };
  int rc = check_paged(cache, n_tokens, n_heads);
  if (rc) return rc;
  if (act_dtype != JERO_F32 && act_dtype != JERO_F16)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "activations must be JERO_F32 or JERO_F16");
  if (act_dtype == JERO_F16 && cache->kv_dtype != JERO_KV_F16)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "f16 activations need an f16 cache");
  if (!q_dev || !out_dev) return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  if ((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev)) & 15u)
    return bad(JERO_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
  if (q_stride < int64_t(n_heads) * cache->head_dim || out_stride < int64_t(n_heads) * cache->head_dim)
    return bad(JERO_ERR_TENSOR_BOUNDS, "rows overlap: a stride is below its row's length");
  if (q_stride % 8 || out_stride % 8) return bad(JERO_ERR_INVALID_ARGUMENT, "strides must be multiples of 8 elements");
  if (!std::isfinite(scale)) return bad(JERO_ERR_INVALID_ARGUMENT, "scale must be finite");
  const PagedPlan p = paged_plan(cache, act_dtype == JERO_F16, n_tokens, n_heads);
  size_t ml = 0;
  const size_t need = part_bytes(p, n_tokens, n_heads, cache->head_dim, &ml);
  if (need) {
    if (!workspace_dev) {
      if ((rc = workspace(need, &workspace_dev))) return rc;
    } else if (workspace_bytes < need) {
      return fail(JERO_ERR_TENSOR_BOUNDS, "paged_attention: workspace of " + std::to_string(workspace_bytes) +
                                              " bytes, need " + std::to_string(need));
    } else if (reinterpret_cast<uintptr_t>(workspace_dev) & 255u) {
      return bad(JERO_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    }
  }
  PagedCall c{};
  c.k = cache->k_dev, c.v = cache->v_dev;
  c.table = cache->table_dev, c.lens = cache->lens_dev, c.starts = cache->starts_dev, c.shared = cache->shared_dev;
  c.table_stride = cache->table_stride;
  c.q_stride = q_stride, c.out_stride = out_stride;
  c.n_blocks = uint32_t(cache->n_blocks);
  c.n_seqs = int(cache->n_seqs), c.n_tokens = int(n_tokens), c.max_len = int(cache->max_len);
  c.shared_len = int(std::min<int64_t>(cache->shared_blocks * cache->block_size, cache->max_len));
  c.shared_blocks = int(cache->shared_blocks);
  c.shift = __builtin_ctz(unsigned(cache->block_size));
  c.heads = n_heads, c.kv_heads = cache->n_heads_kv, c.group = n_heads / cache->n_heads_kv, c.dim = cache->head_dim;
  c.scale = scale;
  float* part_o = static_cast<float*>(workspace_dev);
  float2* part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace_dev) + ml);
  const bool x16 = act_dtype == JERO_F16, kv16 = cache->kv_dtype == JERO_KV_F16;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int hd = head_width(c.dim);
  rc = (hd == 64 ? paged_attend_64 : hd == 128 ? paged_attend_128 : paged_attend_256)(c, p, x16, kv16, q_dev, out_dev, part_o,
                                                                                    part_ml, s);
  if (rc || p.parts == 1) return rc;
  if (x16) launch_merge<_Float16>(c, p, out_dev, part_o, part_ml, s);
  else launch_merge<float>(c, p, out_dev, part_o, part_ml, s);
  return check_launch("paged_attention merge");
}
