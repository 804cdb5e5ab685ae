// paged.hip -- a serving step over a paged key/value cache: block tables and slots from the requests'
// lengths, and the step's rows rotated and stored.
#include <cmath>

#include "jero_common.h"
#include "runtime.h"

namespace jero {

// ---------------------------------------------------------------- block tables and slots

struct BlockPool {
  int32_t *table, *free_ids;
  const int32_t *lens, *owned, *n_free, *asked, *drop;
  int32_t *lens_out, *owned_out, *n_free_out, *starts, *granted, *positions;
  int64_t* slots;
  int64_t table_stride, n_blocks;
  int n_seqs, capacity, shared, shift, n_tokens;
};

// What the second part wants of a request: its positions and blocks before the call, and the blocks taken before it.
struct Request {
  int len, owned, taken;  // len -1: not granted
};
// The stack: ids before, and with those given back; then how many are taken and given back in all.
struct Stack {
  int before, top, taken, back;
};
// The workspace's arrays: a request's, and the sums of blocks given back before each.
struct ExtendSpace {
  Request* r;
  int32_t* back;
  Stack* st;
};

constexpr int kExtendThreads = 1024, kExtendWaves = kExtendThreads / kWave;

template <typename T>
__device__ __forceinline__ T wave_scan(T v, int lane) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const T o = __shfl_up(v, off, kWave);
    if (lane >= off) v += o;
  }
  return v;
}

struct Held {
  int len, owned, need, back, tokens;
  bool ends, fits;
};
__device__ __forceinline__ Held held_by(const BlockPool& p, int s) {
  Held h;
  const int asked = p.asked[s];
  h.ends = asked < 0;
  h.tokens = max(asked, 0);
  const int drop = p.drop ? max(p.drop[s], 0) : 0, len = max(p.lens[s], 0);
  h.len = len - min(drop, len);
  h.owned = min(max(p.owned[s], 0), int(p.table_stride));
  const int64_t end = int64_t(h.len) + h.tokens, most = p.table_stride << p.shift;
  h.fits = end <= most;
  const int64_t blocks = (end + (int64_t(1) << p.shift) - 1) >> p.shift;
  h.need = h.tokens > 0 && h.fits ? int(max(blocks - h.owned, int64_t(0))) : 0;
  h.back = h.ends ? max(h.owned - p.shared, 0) : 0;
  return h;
}

// The last of n entries that is not above x (the first is not).
__device__ __forceinline__ int last_not_above(const int32_t* v, int n, int stride, int x) {
  int lo = 0, left = n;
  while (left > 1) {
    const int half = left >> 1;
    if (v[int64_t(lo + half) * stride] <= x) lo += half;
    left -= half;
  }
  return lo;
}

// Id e of those given back, in order.
__device__ __forceinline__ int returned_id(const BlockPool& p, const int32_t* back, int e) {
  const int s = last_not_above(back, p.n_seqs, 1, e);
  return p.table[int64_t(s) * p.table_stride + p.shared + (e - back[s])];
}
// Block i (of all that the call takes, in order): the ids given back stand above those that were there.
__device__ __forceinline__ int taken_id(const BlockPool& p, const int32_t* back, const Stack& st, int i) {
  const int j = st.top - 1 - i;
  return j < st.before ? p.free_ids[j] : returned_id(p, back, j - st.before);
}

// Three sums over the requests (tokens, blocks needed, blocks given back), then each token's place by a search in them.  The
// bytes are few; what bounds it is latencies one after another: a request's counts, the sums, the search, the block's id.
// 64 requests of one token: one launch, 6.5 us; 1500 requests, 281552 tokens, 4395 blocks taken and
// 6016 given back: 9.8 and 10.7 us (64-bit sums in three passes and searches in memory 22.6 and 11.7).

// First part: the sums over the requests, by one workgroup, a request a thread and round.  All that is given back is
// there before the first block is taken, so its sum comes first, from the requests of the first round as they are kept.
__device__ void extend_sums(const BlockPool& p, const ExtendSpace& to, int tid) {
  __shared__ int s_got;
  __shared__ int64_t s_sum[2][3][kExtendWaves], s_back[kExtendWaves];
  const int lane = tid & 63, wv = tid >> 6;
  Held h = {};
  if (tid < p.n_seqs) h = held_by(p, tid);
  int64_t back = h.back;
  for (int s = tid + kExtendThreads; s < p.n_seqs; s += kExtendThreads) back += held_by(p, s).back;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) back += __shfl_xor(back, off, kWave);
  if (lane == 0) s_back[wv] = back;
  if (tid == 0) s_got = 0;
  const int before = min(max(p.n_free[0], 0), p.capacity);
  int top = 0;
  int64_t carry[3] = {0, 0, 0};
  for (int s0 = 0, round = 0; s0 < p.n_seqs; s0 += kExtendThreads, round ^= 1) {
    const int s = s0 + tid;
    const bool on = s < p.n_seqs;
    if (s0) {
      h = Held{};
      if (on) h = held_by(p, s);
    }
    // (tokens in 64 bits: a request may ask for any number; the table's entries, so its blocks, are below 2^31 in all)
    const int64_t w[3] = {wave_scan(int64_t(h.tokens), lane), wave_scan(h.need, lane), wave_scan(h.back, lane)};
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (lane == 63) s_sum[round][i][wv] = w[i];
    __syncthreads();
    if (s0 == 0) {
      int64_t all = before;
#pragma unroll
      for (int i = 0; i < kExtendWaves; i++) all += s_back[i];
      top = int(min(all, int64_t(p.capacity)));
    }
    int64_t sum[3];
#pragma unroll
    for (int i = 0; i < 3; i++) {
      // (16 waves' sums, a lane each)
      const int64_t v = s_sum[round][i][lane & (kExtendWaves - 1)];
      int64_t below = (lane & (kExtendWaves - 1)) < wv ? v : 0, all = v;
#pragma unroll
      for (int off = 1; off < kExtendWaves; off <<= 1) below += __shfl_xor(below, off, kWave), all += __shfl_xor(all, off, kWave);
      sum[i] = carry[i] + below + w[i];
      carry[i] += all;
    }
    const bool granted = h.fits && (h.need == 0 || sum[1] <= top);
    if (on) {
      p.starts[s] = int(min(sum[0] - h.tokens, int64_t(INT32_MAX)));
      to.r[s] = Request{granted ? h.len : -1, h.owned, int(sum[1] - h.need)};
      to.back[s] = int(sum[2] - h.back);
      p.lens_out[s] = h.ends ? 0 : granted ? h.len + h.tokens : h.len;
      p.owned_out[s] = h.ends ? 0 : granted ? h.owned + h.need : h.owned;
      if (p.granted) p.granted[s] = granted;
    }
    // the needs' sums do not fall, so what is taken is the last granted one's
    const uint64_t some = __ballot(on && granted && h.need > 0);
    if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&s_got, int(sum[1]));
  }
  __syncthreads();
  if (tid == 0) {
    p.starts[p.n_seqs] = int(min(carry[0], int64_t(INT32_MAX)));
    *to.st = Stack{before, top, s_got, int(carry[2])};
    p.n_free_out[0] = top - s_got;
  }
}

// Second part: each token's position and slot, the blocks given back, and those taken.  starts and back may be copies.
__device__ void extend_rows(const BlockPool& p, const Request* r, const int32_t* starts, const int32_t* back, const Stack& st,
                            int at, int step) {
  const int total = starts[p.n_seqs], mask = (1 << p.shift) - 1;
  for (int64_t item = at; item < int64_t(p.n_tokens) + st.back + st.taken; item += step) {
    if (item < p.n_tokens) {
      const int i = int(item);
      int pos = -1;
      int64_t slot = -1;
      if (i < total) {
        const int s = last_not_above(starts, p.n_seqs, 1, i);
        const Request q = r[s];
        if (q.len >= 0) {
          pos = q.len + (i - starts[s]);
          const int c = pos >> p.shift;
          const int id = c < q.owned ? p.table[int64_t(s) * p.table_stride + c] : taken_id(p, back, st, q.taken + c - q.owned);
          if (uint32_t(id) < uint64_t(p.n_blocks)) slot = (int64_t(id) << p.shift) + (pos & mask);
        }
      }
      p.positions[i] = pos;
      p.slots[i] = slot;
    } else if (item < int64_t(p.n_tokens) + st.back) {
      const int e = int(item - p.n_tokens);
      if (e < p.capacity - st.before) p.free_ids[st.before + e] = returned_id(p, back, e);
    } else {
      const int k = int(item - p.n_tokens - st.back), s = last_not_above(&r[0].taken, p.n_seqs, sizeof(Request) / 4, k);
      p.table[int64_t(s) * p.table_stride + r[s].owned + (k - r[s].taken)] = taken_id(p, back, st, k);
    }
  }
}

// One launch, its arrays in LDS, up to this many requests and tokens.  (The host does not know how many blocks are given back,
// which that one workgroup does too: 1024 requests that end with 512 blocks each take 391 us, by two launches 98; 128 of them
// 54 and 22; where none end 7.8 and 12.4.)
constexpr int kExtendSeqs = 1024, kExtendTokens = 4096;
// Requests whose starts and sums of blocks given back the second launch's workgroups copy to LDS: 11 steps of a search
// there for 1500 requests, 11 times the memory's latency otherwise.
constexpr int kExtendCopied = 4096;

__global__ void __launch_bounds__(kExtendThreads) extend_small_kernel(BlockPool p) {
  __shared__ Request s_r[kExtendSeqs];
  __shared__ int32_t s_back[kExtendSeqs];
  __shared__ Stack s_st;
  extend_sums(p, ExtendSpace{s_r, s_back, &s_st}, threadIdx.x);
  __syncthreads();
  extend_rows(p, s_r, p.starts, s_back, s_st, threadIdx.x, kExtendThreads);
}
__global__ void __launch_bounds__(kExtendThreads) extend_sums_kernel(BlockPool p, ExtendSpace to) {
  extend_sums(p, to, threadIdx.x);
}
template <bool COPIED>
__global__ void __launch_bounds__(256) extend_rows_kernel(BlockPool p, ExtendSpace from) {
  if constexpr (COPIED) {
    __shared__ int32_t s_starts[kExtendCopied + 1], s_back[kExtendCopied];
    for (int i = threadIdx.x; i <= p.n_seqs; i += 256) s_starts[i] = p.starts[i];
    for (int i = threadIdx.x; i < p.n_seqs; i += 256) s_back[i] = from.back[i];
    __syncthreads();
    extend_rows(p, from.r, s_starts, s_back, *from.st, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
  } else {
    extend_rows(p, from.r, p.starts, from.back, *from.st, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
  }
}

// ---------------------------------------------------------------- rotation and storing

template <typename X>
__device__ __forceinline__ void row_load4(const X* p, float* v);
template <>
__device__ __forceinline__ void row_load4<float>(const float* p, float* v) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
template <>
__device__ __forceinline__ void row_load4<_Float16>(const _Float16* p, float* v) {
  const h4v a = *reinterpret_cast<const h4v*>(p);
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = float(a[e]);
}
__device__ __forceinline__ void row_store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void row_store4(_Float16* p, const float* v) {
  h4v a;
#pragma unroll
  for (int e = 0; e < 4; e++) a[e] = _Float16(v[e]);
  *reinterpret_cast<h4v*>(p) = a;
}

struct AppendArgs {
  int64_t q_stride, k_stride, v_stride, q_out_stride, n_slots;
  const int32_t* positions;
  const int64_t* slots;
  const float *q_norm, *k_norm;
  float eps;
  int heads, kv_heads, dim;
};

// y_a = m (x_a cos - x_b sin), y_b = m (x_a sin + x_b cos) of a pair (a, b) at position * f.  Bound by the bytes: 12001 tokens
// of 32 + 8 + 8 heads of 128, f16: 295 MB in 50.6 us, 5.8 TB/s; 64 tokens, f32 into f16, both norms: 4.6 us, of which most is
// the chain positions, rows, stores.
// Workgroup (token, run of its rows): LP lanes a row, 8 elements a lane: four pairs of the rotated part (with the
// halves' layout 4 + 4 elements rot / 2 apart), or 8 behind it.  A lane keeps its pairs from row to row, so their
// angles are found once.
template <typename X, typename KV, int LP>
__global__ void __launch_bounds__(256) append_kernel(const X* q, const X* __restrict__ k, const X* __restrict__ v,
                                                     AppendArgs a, jero_rope rope, X* q_out, KV* __restrict__ k_rows,
                                                     KV* __restrict__ v_rows) {
  const int64_t t = blockIdx.x;
  const int u = threadIdx.x % LP, sub = threadIdx.x / LP;
  constexpr int RPB = 256 / LP;
  const int pos = a.positions ? a.positions[t] : 0;
  if (pos < 0) return;
  int64_t slot = a.kv_heads ? a.slots[t] : -1;
  if (uint64_t(slot) >= uint64_t(a.n_slots)) slot = -1;
  const bool on = u < a.dim / 8, turn = u < rope.rot_dim / 8;
  const bool half = turn && rope.layout == JERO_ROPE_HALF;
  const int lo = half ? 4 * u : 8 * u, hi = half ? lo + rope.rot_dim / 2 : lo + 4;
  float c[4], n[4];
  if (turn) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      // the turns are reduced to [-1/2, 1/2] in 64 bits: only the angle within a half turn is in 32
      double x = double(pos) * rope.turns[4 * u + i];
      x -= rint(x);
      sincospif(float(2.0 * x), &n[i], &c[i]);
      c[i] *= rope.magnitude, n[i] *= rope.magnitude;
    }
  }
  const int rows = a.heads + 2 * a.kv_heads;
  for (int r = blockIdx.y * RPB + sub; r < rows; r += gridDim.y * RPB) {
    const bool is_q = r < a.heads, is_k = !is_q && r < a.heads + a.kv_heads;
    const int h = is_q ? r : is_k ? r - a.heads : r - a.heads - a.kv_heads;
    if (!is_q && slot < 0) continue;
    const X* src = (is_q ? q + t * a.q_stride : is_k ? k + t * a.k_stride : v + t * a.v_stride) + int64_t(h) * a.dim;
    float x[8] = {};
    if (on) {
      row_load4<X>(src + (is_q || is_k ? lo : 8 * u), x);
      row_load4<X>(src + (is_q || is_k ? hi : 8 * u + 4), x + 4);
    }
    const float* w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    if (w) {  // (a row's lanes take the same way)
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) sum = fmaf(x[e], x[e], sum);
#pragma unroll
      for (int off = LP / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
      const float f = 1.0f / sqrtf(sum / float(a.dim) + a.eps);
      if (on) {
        float g[8];
        row_load4<float>(w + lo, g);
        row_load4<float>(w + hi, g + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = x[e] * f * g[e];
      }
    }
    if (!on) continue;
    if (turn && (is_q || is_k)) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float p = half ? x[i] : x[2 * i], s = half ? x[4 + i] : x[2 * i + 1];
        const float p1 = p * c[i] - s * n[i], s1 = p * n[i] + s * c[i];
        y[i] = p1, y[4 + i] = s1;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] = half ? y[i] : (i & 1) ? y[4 + i / 2] : y[i / 2];
        x[4 + i] = half ? y[4 + i] : (i & 1) ? y[4 + 2 + i / 2] : y[2 + i / 2];
      }
    }
    if (is_q) {
      X* dst = q_out + t * a.q_out_stride + int64_t(h) * a.dim;
      row_store4(dst + lo, x);
      row_store4(dst + hi, x + 4);
    } else {
      KV* dst = (is_k ? k_rows : v_rows) + (slot * a.kv_heads + h) * a.dim;
      row_store4(dst + (is_k ? lo : 8 * u), x);
      row_store4(dst + (is_k ? hi : 8 * u + 4), x + 4);
    }
  }
}

static bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename X, typename KV>
static void launch_append(const void* q, const void* k, const void* v, const AppendArgs& a, const jero_rope& rope,
                          void* q_out, void* k_rows, void* v_rows, int64_t n_tokens, hipStream_t s) {
  const int units = a.dim / 8, lp = units <= 8 ? 8 : units <= 16 ? 16 : 32;
  const int rows = a.heads + 2 * a.kv_heads, rpb = 256 / lp, most = (rows + rpb - 1) / rpb;
  // few tokens: a token's rows over more workgroups
  int y = int(1024 / (n_tokens < 1024 ? n_tokens : 1024));
  if (y > most) y = most;
  const dim3 grid = {unsigned(n_tokens), unsigned(y), 1};
#define JERO_APPEND(LP)                                                                                             \
  hipLaunchKernelGGL((append_kernel<X, KV, LP>), grid, dim3(256), 0, s, static_cast<const X*>(q), static_cast<const X*>(k), \
                     static_cast<const X*>(v), a, rope, static_cast<X*>(q_out), static_cast<KV*>(k_rows),           \
                     static_cast<KV*>(v_rows))
  if (lp == 8) JERO_APPEND(8);
  else if (lp == 16) JERO_APPEND(16);
  else JERO_APPEND(32);
#undef JERO_APPEND
}

}  // namespace jero

using namespace jero;

extern "C" size_t jero_hip_paged_extend_workspace_bytes(int64_t n_seqs) {
  return n_seqs < 1 || n_seqs > (1 << 19) ? 0 : sizeof(Stack) + size_t(n_seqs) * (sizeof(Request) + 4);
}

extern "C" int jero_hip_paged_extend(const jero_block_pool* pool, const int32_t* new_dev, const int32_t* drop_dev,
                                     int64_t n_tokens, int32_t* starts_dev, int32_t* granted_dev, int32_t* positions_dev,
                                     int64_t* slots_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  auto bad = [](int status, const char* what) { return fail(status, std::string("paged_extend: ") + what); };
  if (!pool || !pool->table_dev || !pool->lens_dev || !pool->owned_dev || !pool->free_dev || !pool->n_free_dev || !new_dev ||
      !starts_dev || !positions_dev || !slots_dev)
    return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  for (const void* p : {static_cast<const void*>(pool->table_dev), static_cast<const void*>(pool->lens_dev),
                        static_cast<const void*>(pool->owned_dev), static_cast<const void*>(pool->free_dev),
                        static_cast<const void*>(pool->n_free_dev), static_cast<const void*>(pool->lens_out_dev),
                        static_cast<const void*>(pool->owned_out_dev), static_cast<const void*>(pool->n_free_out_dev),
                        static_cast<const void*>(new_dev), static_cast<const void*>(drop_dev),
                        static_cast<const void*>(starts_dev), static_cast<const void*>(granted_dev),
                        static_cast<const void*>(positions_dev)})
    if (!aligned(p, 4)) return bad(JERO_ERR_INVALID_ARGUMENT, "arrays must be 4-byte aligned");
  if (!aligned(slots_dev, 8)) return bad(JERO_ERR_INVALID_ARGUMENT, "slots must be 8-byte aligned");
  if (pool->block_size < 1 || pool->block_size > (1 << 20) || (pool->block_size & (pool->block_size - 1)))
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "block_size is not a power of two up to 2^20");
  if (pool->n_seqs < 1 || n_tokens < 1 || pool->table_stride < 1 || pool->n_blocks < 1 || pool->free_capacity < 1)
    return bad(JERO_ERR_TENSOR_BOUNDS, "no sequences, tokens, blocks or free ids");
  if (pool->n_seqs > (1 << 19) || n_tokens > (1 << 24) || pool->n_blocks > INT32_MAX || pool->free_capacity > INT32_MAX ||
      pool->table_stride > INT32_MAX / pool->n_seqs)
    return bad(JERO_ERR_TENSOR_BOUNDS, "more than 2^19 sequences, 2^24 tokens or 2^31 - 1 blocks or table entries");
  if (pool->table_stride * pool->block_size > INT32_MAX)
    return bad(JERO_ERR_CONTEXT_LENGTH_EXCEEDED, "a table row holds more than 2^31 - 1 positions");
  if (pool->shared_blocks < 0 || pool->shared_blocks > pool->table_stride)
    return bad(JERO_ERR_TENSOR_BOUNDS, "shared_blocks is not within a table row");
  BlockPool p{};
  p.table = pool->table_dev;
  p.free_ids = pool->free_dev;
  p.lens = pool->lens_dev;
  p.owned = pool->owned_dev;
  p.n_free = pool->n_free_dev;
  p.asked = new_dev;
  p.drop = drop_dev;
  p.lens_out = pool->lens_out_dev ? pool->lens_out_dev : pool->lens_dev;
  p.owned_out = pool->owned_out_dev ? pool->owned_out_dev : pool->owned_dev;
  p.n_free_out = pool->n_free_out_dev ? pool->n_free_out_dev : pool->n_free_dev;
  p.starts = starts_dev;
  p.granted = granted_dev;
  p.positions = positions_dev;
  p.slots = slots_dev;
  p.table_stride = pool->table_stride;
  p.n_blocks = pool->n_blocks;
  p.n_seqs = int(pool->n_seqs);
  p.capacity = int(pool->free_capacity);
  p.shared = int(pool->shared_blocks);
  p.shift = __builtin_ctz(unsigned(pool->block_size));
  p.n_tokens = int(n_tokens);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.n_seqs <= kExtendSeqs && p.n_tokens <= kExtendTokens) {
    hipLaunchKernelGGL(extend_small_kernel, dim3(1), dim3(kExtendThreads), 0, s, p);
    return check_launch("paged_extend");
  }
  const size_t need = jero_hip_paged_extend_workspace_bytes(pool->n_seqs);
  int rc;
  if (!workspace_dev) {
    if ((rc = workspace(need, &workspace_dev))) return rc;
  } else if (workspace_bytes < need) {
    return bad(JERO_ERR_TENSOR_BOUNDS, "the workspace is too small");
  } else if (!aligned(workspace_dev, 16)) {
    return bad(JERO_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  }
  uint8_t* const at = static_cast<uint8_t*>(workspace_dev);
  const ExtendSpace space{reinterpret_cast<Request*>(at + sizeof(Stack)),
                          reinterpret_cast<int32_t*>(at + sizeof(Stack) + size_t(p.n_seqs) * sizeof(Request)),
                          reinterpret_cast<Stack*>(at)};
  hipLaunchKernelGGL(extend_sums_kernel, dim3(1), dim3(kExtendThreads), 0, s, p, space);
  if ((rc = check_launch("paged_extend"))) return rc;
  const int64_t items = n_tokens > p.n_seqs ? n_tokens : p.n_seqs, blocks = (items + 255) / 256;
  const dim3 grid = {unsigned(blocks < 2048 ? blocks : 2048), 1, 1};
  if (p.n_seqs <= kExtendCopied) hipLaunchKernelGGL((extend_rows_kernel<true>), grid, dim3(256), 0, s, p, space);
  else hipLaunchKernelGGL((extend_rows_kernel<false>), grid, dim3(256), 0, s, p, space);
  return check_launch("paged_extend rows");
}

extern "C" int jero_hip_rope_init(jero_rope* rope, int rot_dim, int layout, double theta, int scaling, double factor,
                                  double original_len, double low, double high) {
  auto bad = [](int status, const char* what) { return fail(status, std::string("rope_init: ") + what); };
  if (!rope) return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  if (rot_dim < 8 || rot_dim % 8 || rot_dim > 256)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "rot_dim is not a multiple of 8 up to 256");
  if (layout != JERO_ROPE_HALF && layout != JERO_ROPE_INTERLEAVED)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "layout must be JERO_ROPE_HALF or JERO_ROPE_INTERLEAVED");
  if (scaling < JERO_ROPE_NONE || scaling > JERO_ROPE_WAVELENGTH)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "unknown scaling");
  if (!(theta > 1.0) || !std::isfinite(theta)) return bad(JERO_ERR_INVALID_ARGUMENT, "theta must be above 1 and finite");
  if (scaling != JERO_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
    return bad(JERO_ERR_INVALID_ARGUMENT, "factor must be at least 1 and finite");
  const bool ramp = scaling == JERO_ROPE_YARN || scaling == JERO_ROPE_WAVELENGTH;
  if (ramp) {
    if (!(original_len >= 1.0) || !std::isfinite(original_len))
      return bad(JERO_ERR_INVALID_ARGUMENT, "original_len must be at least 1 and finite");
    if (low == 0.0) low = 1.0;
    if (high == 0.0) high = scaling == JERO_ROPE_YARN ? 32.0 : 4.0;
    if (!(low > 0.0) || !(high > low) || !std::isfinite(high))
      return bad(JERO_ERR_INVALID_ARGUMENT, "low must be above 0 and high above low");
  }
  constexpr double kTurn = 6.283185307179586476925;
  *rope = jero_rope{};
  rope->magnitude = 1.0f;
  rope->rot_dim = rot_dim;
  rope->layout = layout;
  if (scaling == JERO_ROPE_NTK) theta *= std::pow(factor, double(rot_dim) / (rot_dim - 2));
  if (scaling == JERO_ROPE_YARN) rope->magnitude = float(0.1 * std::log(factor) + 1.0);
  double lo = 0, hi = 0;
  if (scaling == JERO_ROPE_YARN) {
    auto pair = [&](double turns) { return rot_dim * std::log(original_len / (kTurn * turns)) / (2.0 * std::log(theta)); };
    lo = std::fmax(std::floor(pair(high)), 0.0);
    hi = std::fmin(std::ceil(pair(low)), rot_dim - 1.0);
  }
  for (int i = 0; i < rot_dim / 2; i++) {
    double f = std::pow(theta, -2.0 * i / rot_dim);
    if (scaling == JERO_ROPE_LINEAR) f /= factor;
    if (ramp) {
      double r = scaling == JERO_ROPE_YARN ? (i - lo) / std::fmax(hi - lo, 0.001)
                                           : (original_len * f / kTurn - low) / (high - low);
      r = std::fmin(std::fmax(r, 0.0), 1.0);
      const double stretched = scaling == JERO_ROPE_YARN ? r : 1.0 - r;
      f = f / factor * stretched + f * (1.0 - stretched);
    }
    rope->turns[i] = f / kTurn;
  }
  return JERO_OK;
}

extern "C" int jero_hip_paged_append(int act_dtype, const void* q_dev, int64_t q_stride, const void* k_dev,
                                     int64_t k_stride, const void* v_dev, int64_t v_stride, int64_t n_tokens, int n_heads,
                                     int n_heads_kv, int head_dim, const int32_t* positions_dev, const int64_t* slots_dev,
                                     const jero_rope* rope, const float* q_norm_dev, const float* k_norm_dev, float eps,
                                     void* q_out_dev, int64_t q_out_stride, void* k_rows_dev, void* v_rows_dev, int kv_dtype,
                                     int64_t n_slots, void* stream) {
  auto bad = [](int status, const char* what) { return fail(status, std::string("paged_append: ") + what); };
  if (act_dtype != JERO_F32 && act_dtype != JERO_F16)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "activations must be JERO_F32 or JERO_F16");
  if (kv_dtype != JERO_KV_F32 && kv_dtype != JERO_KV_F16)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "kv_dtype must be JERO_KV_F32 or JERO_KV_F16");
  if (n_heads < 0 || n_heads_kv < 0 || n_heads + int64_t(n_heads_kv) < 1) return bad(JERO_ERR_TENSOR_BOUNDS, "no heads");
  if (n_heads > 1024 || n_heads_kv > 1024) return bad(JERO_ERR_CAPABILITY_MISMATCH, "more than 1024 heads");
  if (head_dim < 8 || head_dim % 8 || head_dim > 256)
    return bad(JERO_ERR_CAPABILITY_MISMATCH, "head_dim is not a multiple of 8 up to 256");
  if (n_tokens < 1 || n_tokens >= (1 << 24))  // (256 threads each, and a launch has fewer than 2^32)
    return bad(JERO_ERR_TENSOR_BOUNDS, "tokens must be 1 to 2^24 - 1");
  if (n_heads && (!q_dev || !q_out_dev)) return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  if (n_heads_kv && (!k_dev || !v_dev || !k_rows_dev || !v_rows_dev || !slots_dev))
    return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  if (rope && !positions_dev) return bad(JERO_ERR_INVALID_ARGUMENT, "a rotation needs positions");
  if (n_heads && (!aligned(q_dev, 16) || !aligned(q_out_dev, 16)))
    return bad(JERO_ERR_INVALID_ARGUMENT, "q and q_out must be 16-byte aligned");
  if (n_heads_kv && (!aligned(k_dev, 16) || !aligned(v_dev, 16) || !aligned(k_rows_dev, 16) || !aligned(v_rows_dev, 16)))
    return bad(JERO_ERR_INVALID_ARGUMENT, "keys, values and pools must be 16-byte aligned");
  if (!aligned(positions_dev, 4) || !aligned(slots_dev, 8) || !aligned(q_norm_dev, 16) || !aligned(k_norm_dev, 16))
    return bad(JERO_ERR_INVALID_ARGUMENT, "positions, slots and norms must be aligned to 4, 8 and 16 bytes");
  const int64_t wide = int64_t(n_heads) * head_dim, wide_kv = int64_t(n_heads_kv) * head_dim;
  if ((n_heads && (q_stride < wide || q_out_stride < wide)) || (n_heads_kv && (k_stride < wide_kv || v_stride < wide_kv)))
    return bad(JERO_ERR_TENSOR_BOUNDS, "rows overlap: a stride is below its row's length");
  if ((n_heads && (q_stride % 8 || q_out_stride % 8)) || (n_heads_kv && (k_stride % 8 || v_stride % 8)))
    return bad(JERO_ERR_INVALID_ARGUMENT, "strides must be multiples of 8 elements");
  if (n_heads && q_out_dev == q_dev && n_tokens > 1 && q_out_stride != q_stride)
    return bad(JERO_ERR_INVALID_ARGUMENT, "queries rotated in place need one stride");
  if (n_heads_kv && n_slots < 1) return bad(JERO_ERR_TENSOR_BOUNDS, "no slots");
  if ((q_norm_dev || k_norm_dev) && !(eps >= 0.f && std::isfinite(eps)))
    return bad(JERO_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  jero_rope none{};
  if (rope) {
    if (rope->rot_dim < 8 || rope->rot_dim % 8 || rope->rot_dim > head_dim)
      return bad(JERO_ERR_TENSOR_BOUNDS, "the rotation is wider than a head");
    if (rope->layout != JERO_ROPE_HALF && rope->layout != JERO_ROPE_INTERLEAVED)
      return bad(JERO_ERR_CAPABILITY_MISMATCH, "layout must be JERO_ROPE_HALF or JERO_ROPE_INTERLEAVED");
  }
  const AppendArgs a{q_stride, k_stride, v_stride, q_out_stride, n_slots, positions_dev, slots_dev, q_norm_dev,
                     k_norm_dev, eps, n_heads, n_heads_kv, head_dim};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const jero_rope& r = rope ? *rope : none;
  const bool x16 = act_dtype == JERO_F16, kv16 = kv_dtype == JERO_KV_F16;
  if (x16 && kv16) launch_append<_Float16, _Float16>(q_dev, k_dev, v_dev, a, r, q_out_dev, k_rows_dev, v_rows_dev, n_tokens, s);
  else if (x16) launch_append<_Float16, float>(q_dev, k_dev, v_dev, a, r, q_out_dev, k_rows_dev, v_rows_dev, n_tokens, s);
  else if (kv16) launch_append<float, _Float16>(q_dev, k_dev, v_dev, a, r, q_out_dev, k_rows_dev, v_rows_dev, n_tokens, s);
  else launch_append<float, float>(q_dev, k_dev, v_dev, a, r, q_out_dev, k_rows_dev, v_rows_dev, n_tokens, s);
  return check_launch("paged_append");
}
