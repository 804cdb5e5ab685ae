// mla.h -- latent attention over a paged cache: what its kernels and launchers share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jero_common.h"
#include "runtime.h"

namespace jero {

constexpr int kMlaMaxRank = 512;
constexpr int kMlaMaxRope = 64;

// A jero_latent_cache as the kernels take it.
struct LatentCache {
  const void* rows;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
  int64_t table_stride;
  uint32_t n_blocks;
  int n_seqs, n_tokens;
  int max_len;
  int shift;  // log2 of the block size
  int rank, rope, width;
};

// Turns of pair i per position, theta^(-2i / rope) / 2 pi, in 64 bits: at position 131072 an angle in
// 32 bits is off by up to 0.008.  on = 0: rows come rotated.
struct MlaRope {
  double turns[kMlaMaxRope / 2];
  int on;
};

// (cos, sin) of pair i at pos: the turns are reduced to [-1/2, 1/2] in 64 bits, so that only the last
// step, of an angle within a half turn, is in 32.
__device__ __forceinline__ float2 mla_cos_sin(const MlaRope& rope, int i, int pos) {
  double t = double(pos) * rope.turns[i];
  t -= rint(t);
  float s, c;
  sincospif(float(2.0 * t), &s, &c);
  return make_float2(c, s);
}

// The sequence and position of token row t, found by the whole wave: the sequence is the last whose
// start is not behind t, and the starts do not decrease, so counting them is enough.  False for rows
// of no sequence.
__device__ __forceinline__ bool mla_locate(const LatentCache& c, int t, int lane, int& seq, int& pos) {
  if (!c.starts) {
    seq = t;
    pos = c.lens[t] - 1;
    return true;
  }
  int count = 0;
  for (int j0 = 0; j0 <= c.n_seqs; j0 += kWave) {
    const int j = j0 + lane;
    const bool below = j <= c.n_seqs && c.starts[min(j, c.n_seqs)] <= t;
    const int n = __popcll(__ballot(below));
    count += n;
    if (n < kWave) break;
  }
  seq = count - 1;
  if (seq < 0 || seq >= c.n_seqs) return false;
  const int first = c.starts[seq], end = c.starts[seq + 1];
  pos = int(int64_t(c.lens[seq]) - end + t);
  return t >= first;
}

// Offset in elements of the cache row of (seq, pos), 0 <= pos < max_len; -1 for a block that is none.
__device__ __forceinline__ int64_t mla_row(const LatentCache& c, int seq, int pos) {
  const uint32_t b = uint32_t(c.table[seq * c.table_stride + (pos >> c.shift)]);
  if (b >= c.n_blocks) return -1;
  return ((int64_t(b) << c.shift) + (pos & ((1 << c.shift) - 1))) * c.width;
}

int mla_check_cache(const jero_latent_cache* cache, int64_t n_tokens, int act_dtype, const char* what);
LatentCache mla_cache_of(const jero_latent_cache* cache, int64_t n_tokens);
int mla_rope_of(float theta, int rope_dim, MlaRope* out);
int mla_check_attention(const jero_latent_cache* cache, int act_dtype, const void* q, int64_t q_stride,
                        int64_t n_tokens, int n_heads, int nope, int v, const void* w0, const void* w1, float scale,
                        const void* out, int64_t out_stride, const char* what);

}  // namespace jero
