// mla.h -- latent attention over a paged cache: what its kernels and launchers share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jero_common.h"
#include "runtime.h"

namespace jero {

constexpr int kMlaMaxRank = 512;
constexpr int kMlaMaxRope = 64;

// Softmax numerators go into the f16 products (and the totals) 2^Lift above 2^(score - maximum), and a row's
// accumulators are rescaled once its maximum grew by more than 2^Grow: none is above 2^15, and f16's last place,
// 2^-24, is at most 2^(-24 - Lift) of the row's largest.  Not lifted, 6 % are lost of 8192 positions 16 nats below a
// peak (9e-4 of the row), and all of them at 17.4 nats.  The absorbed form's runs are short and rescaling 16 heads'
// 512 columns is dear: one token of 131072 positions takes 107 us in all with Grow 6, 109 with 5, 111 with 4 (106
// with 8), 64 f16 sequences 116, 119, 123 (115).  The expanded form's time is the same.
constexpr float kAttendLift = 9.f, kAttendGrow = 6.f, kFlashLift = 11.f, kFlashGrow = 4.f;

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

// The call's token rows that belong to a sequence, [lo, hi): the others' memory need not be there.
__device__ __forceinline__ void mla_owned(const LatentCache& c, int& lo, int& hi) {
  lo = c.starts ? max(c.starts[0], 0) : 0;
  hi = c.starts ? min(c.starts[c.n_seqs], c.n_tokens) : c.n_tokens;
}

// Position of token row t of a sequence that ends before row `end` with `len` positions; far below 0 it stays there.
__device__ __forceinline__ int mla_position(int len, int end, int t) {
  return int(max(int64_t(len) - end + t, int64_t(-(1 << 30))));
}

// The sequence and position of token row t, found by the whole wave: the sequence is the last whose
// start is not behind t, and the starts do not decrease, so counting them is enough: 64 spread over those
// left at a time.  False for rows of no sequence.
__device__ __forceinline__ bool mla_locate(const LatentCache& c, int t, int lane, int& seq, int& pos) {
  if (!c.starts) {
    seq = t;
    pos = mla_position(c.lens[t], 1, 0);
    return true;
  }
  int count = 0, left = c.n_seqs + 1;  // starts below `count` are not behind t, those from count + left on are
  while (left > 0) {
    const int step = (left + kWave - 1) / kWave, j = count + lane * step + step - 1;  // a step's last
    const int n = __popcll(__ballot(j < count + left && c.starts[min(j, c.n_seqs)] <= t));
    const int past = n * step;
    left = min(step - 1, left - past);
    count += past;
  }
  seq = count - 1;
  if (seq < 0 || seq >= c.n_seqs) return false;
  const int first = c.starts[seq], end = c.starts[seq + 1];
  pos = mla_position(c.lens[seq], end, t);
  return t >= first;
}

// Offset in elements of the cache row of (seq, pos), 0 <= pos < max_len; -1 for a block that is none.
__device__ __forceinline__ int64_t mla_row(const LatentCache& c, int seq, int pos) {
  const uint32_t b = uint32_t(c.table[seq * c.table_stride + (pos >> c.shift)]);
  if (b >= c.n_blocks) return -1;
  return ((int64_t(b) << c.shift) + (pos & ((1 << c.shift) - 1))) * c.width;
}

// ---------------------------------------------------------------- matrix cores, LDS

typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f4_t mfma(h8_t a, h8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// x as two f16 parts, hi + lo = x to 22 bits.
__device__ __forceinline__ void split2(float x, _Float16& hi, _Float16& lo) {
  hi = _Float16(x);
  lo = _Float16(x - float(hi));
}

template <typename X>
__device__ __forceinline__ void load8(const X* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<_Float16>(const _Float16* p, float (&v)[8]) {
  const h8_t a = *reinterpret_cast<const h8_t*>(p);
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = float(a[e]);
}

// Over lanes l, l ^ 16, l ^ 32, l ^ 48: each swap leaves a value and its partner in the two results.
__device__ __forceinline__ float max_over_groups(float v) {
  const uint32_t x = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// 16 bytes a lane straight from global memory to LDS, lane l's to base + 16 l: the loads in flight take no
// registers.  The compiler does not know of these loads; dma_wait waits for the wave's own but the last N, and
// a barrier then shows them to the others.
__device__ __forceinline__ void dma_row(const void* row, uint32_t lane_bytes, uint32_t lds) {  // uniform row
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(lane_bytes), "s"(row)
               : "memory");
}
__device__ __forceinline__ void dma_lanes(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}
template <int N>
__device__ __forceinline__ void dma_wait() {
  static_assert(N < 64, "the counter's range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) s4_t lds_s4;

// The swap of a row's 16-byte chunks in LDS (chunk k of row r sits at k ^ swap8(r)) with which neither 8 rows'
// reads of one chunk nor a transposing read's 32 bytes of 4 rows meet on a bank, for rows of a multiple of 128 bytes;
// rows of 64 bytes have 4 chunks to swap.
__host__ __device__ __forceinline__ constexpr int swap8(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }
__host__ __device__ __forceinline__ constexpr int swap4(int r) { return (r >> 1) & 3; }

int mla_check_cache(const jero_latent_cache* cache, int64_t n_tokens, int act_dtype, const char* what);
LatentCache mla_cache_of(const jero_latent_cache* cache, int64_t n_tokens);
int mla_rope_of(float theta, int rope_dim, MlaRope* out);
int mla_check_attention(const jero_latent_cache* cache, int act_dtype, const void* q, int64_t q_stride,
                        int64_t n_tokens, int n_heads, int nope, int v, const void* w0, const void* w1, float scale,
                        const void* out, int64_t out_stride, const char* what);

}  // namespace jero
