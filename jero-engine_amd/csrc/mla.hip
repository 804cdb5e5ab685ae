// mla.hip -- latent attention over a paged cache: appending rows, and the absorbed form.
#include "mla.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace jero {

// ---------------------------------------------------------------- append

// One wave per token row: lane l holds elements 8l .. 8l + 7 of the latent, the first rope / 2 lanes a
// pair of the key part each.  The sum of squares is f32; the row is rounded once, to the cache's type.
// VEC: the rows of x are 16-byte aligned, and are read so (stores always are: 8-element rows of the pool).  What
// a row of some sequence needs is on its way before its place is looked up.
//
// Bound by its bytes, for a decode step by the launch: 16638 rows of 576 f16 values take 11.0 us (3.5 TB/s; a large
// copy 4.6), 64 rows 3.3 us; one value a lane and load took 30 us.
template <typename X, typename KV, bool VEC>
__global__ void __launch_bounds__(256) mla_append_kernel(LatentCache c, const X* __restrict__ x, int64_t x_stride,
                                                         const float* __restrict__ norm, float eps, MlaRope rope) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  int lo, hi;
  mla_owned(c, lo, hi);
  if (t < lo || t >= hi) return;
  const X* xr = x + t * x_stride;
  const int k = min(8 * lane, c.rank - 8), i = min(lane, c.rope / 2 - 1);
  float v[8], w[8];
  if constexpr (VEC) {
    load8<X>(xr + k, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = float(xr[k + e]);
  }
  if (norm) {
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = norm[k + e];
  }
  const float a = float(xr[c.rank + 2 * i]), b = float(xr[c.rank + 2 * i + 1]);
  int seq, pos;
  if (!mla_locate(c, t, lane, seq, pos) || pos < 0 || pos >= c.max_len) return;
  const int64_t at = mla_row(c, seq, pos);
  if (at < 0) return;
  KV* row = static_cast<KV*>(const_cast<void*>(c.rows)) + at;
  const bool in = 8 * lane < c.rank;
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) ss += in ? v[e] * v[e] : 0.f;
    ss = wave_sum_dpp(ss);
    const float inv = 1.0f / sqrtf(ss / float(c.rank) + eps);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = v[e] * inv * w[e];
  }
  if (in) {
    if constexpr (sizeof(KV) == 4) {
      reinterpret_cast<float4*>(row + k)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(row + k)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      h8_t y;
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = _Float16(v[e]);
      *reinterpret_cast<h8_t*>(row + k) = y;
    }
  }
  if (lane < c.rope / 2) {
    const float2 cs = rope.on ? mla_cos_sin(rope, lane, pos) : make_float2(1.f, 0.f);
    const float y = a * cs.x - b * cs.y, z = a * cs.y + b * cs.x;
    if constexpr (sizeof(KV) == 4) {
      *reinterpret_cast<float2*>(row + c.rank + 2 * lane) = make_float2(y, z);
    } else {
      typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
      *reinterpret_cast<h2_t*>(row + c.rank + 2 * lane) = h2_t{_Float16(y), _Float16(z)};
    }
  }
}

// ---------------------------------------------------------------- absorbed attention
//
// Three launches.  mla_absorb_kernel makes the absorbed queries q' = [q_n W_uk | rotated q_p] and the
// plan; mla_attend_kernel reads every cache row once for up to 64 heads (128 with f16 activations), with a
// running maximum and sum, and leaves one partial row per (run of tiles, token, head); mla_values_kernel
// merges a token's partials and applies W_uv.
//
// The plan cuts the tiles of all tokens, one after the other, into equal runs, one per workgroup and
// group of heads, so that ragged lengths fill the chip: with splits of equal length per token, 32
// sequences of 900 to 6000 positions leave half the workgroups short.  Run w of token t writes partial
// w + t: along the runs either w or t grows, so the number names the pair.

constexpr int kMlaRuns = 256;  // workgroups of the attend kernel: one per CU, its tiles fill the LDS
constexpr int kMlaTile = 32;   // positions a step
constexpr int kMlaBegin = 3;   // what beginning an item takes, in steps

struct MlaPlan {
  int* prefix;  // [T + 1] tiles before each token
  int* seq;     // [T] sequence, -1 for a row of none
  int* end;     // [T] positions attended to, an item's by its last token
  int* item;    // [T] the item's first token
};

// An item: up to `share` tokens of a sequence, one after the other, whose heads attend to its rows together, token
// after token (so that drafted tokens read them once; 1: each token by itself).  Its units are its first token's.
// Number of an item, no two alike and growing: along a sequence first / share grows, from one to the next seq does.
__device__ __forceinline__ int mla_item(int share, int seq, int first) { return share > 1 ? seq + first / share : first; }
__device__ __forceinline__ int mla_item_first(const LatentCache& c, int share, int seq, int t) {
  return share > 1 ? t - (t - max(c.starts[seq], 0)) % share : t;
}
__device__ __forceinline__ int mla_item_tokens(const LatentCache& c, int share, int seq, int first) {
  return share > 1 ? min(share, min(c.starts[seq + 1], c.n_tokens) - first) : 1;
}

// Sequence and position of token t by one thread (mla_locate is a wave's).
__device__ __forceinline__ bool mla_locate_thread(const LatentCache& c, int t, int& seq, int& pos) {
  if (!c.starts) {
    seq = t;
    pos = mla_position(c.lens[t], 1, 0);
    return true;
  }
  int lo = 0, hi = c.n_seqs + 1;  // starts below lo are <= t, those from hi on are not
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c.starts[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  seq = lo - 1;
  if (seq < 0 || seq >= c.n_seqs) return false;
  pos = mla_position(c.lens[seq], c.starts[seq + 1], t);
  return true;
}

// The absorbed queries, as the attend kernel's waves take them: for each token and 16 heads, and each 32 of
// the padded columns (rt for the latent, then the key part's), the 64 lanes' 8 halves of an MFMA operand (lane
// 16 g + i: head i, columns 8g ..); the upper parts, and `plane` further on the lower ones.  A head's row is
// brought near 1 by a power of two, so that its parts stay within f16's range; factor holds what is to be
// multiplied onto its scores, in log2.
struct MlaQueries {
  _Float16* parts;
  float* factor;  // [T][heads to whole 16s]
  int64_t plane;
  int rt, kt;     // padded latent columns, 32s of all columns
};

// Blocks that read the same head's weights for different tokens, on one XCD (blocks go round the 8) and one
// after the other, so that all but the first find them in its L2: block b of `per` blocks a head.
__device__ __forceinline__ bool mla_head_block(int b, int nh, int per, int& h, int& part) {
  h = (b / (8 * per)) * 8 + (b & 7);
  part = (b >> 3) % per;
  return h < nh;
}
static unsigned mla_head_blocks(int nh, int per) { return unsigned((nh + 7) / 8 * 8) * unsigned(per); }
// The same with 8 heads on one XCD, where what they write shares lines.
__device__ __forceinline__ bool mla_head8_block(int b, int nh, int per, int& h, int& part) {
  const int slot = b >> 3, in = slot % (8 * per);
  h = ((slot / (8 * per)) * 8 + (b & 7)) * 8 + in / per;
  part = in % per;
  return h < nh;
}
static unsigned mla_head8_blocks(int nh, int per) { return unsigned((nh + 63) / 64 * 64) * unsigned(per); }

// A block per head and 16 tokens, and one more for the plan.  The 8 waves take the head's rows of W_uk^T by 16; a
// thread rotates a pair of the key part; the row's largest value is the scale of its parts.  Bound by the way of
// one block's loads, a chain of memory latencies: 9.5 us for one token of 128 heads (16.8 MB of weights), 18 us for 64
// (f16; the weights come from L2 for 16 tokens each).
template <typename X, int NT>
__global__ void __launch_bounds__(512) mla_absorb_kernel(LatentCache c, const X* __restrict__ q, int64_t q_stride, int nh,
                                                         int nope, const _Float16* __restrict__ k_b, MlaRope rope,
                                                         float scale, MlaQueries qa, MlaPlan plan, int share) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  if (blockIdx.x + 1 < gridDim.x) {
    int h, t0;
    if (!mla_head8_block(blockIdx.x, nh, (c.n_tokens + 15) / 16, h, t0)) return;
    t0 *= 16;
    int lo, hi;
    mla_owned(c, lo, hi);
    constexpr int NR = kMlaMaxRank / 128;  // 16s of rows a wave
    __shared__ float s_max[8][16];
    __shared__ uint32_t s_key[16];
    __shared__ int s_ex[16], s_first[16];
    const int g = lane >> 4, col = lane & 15;
    // everything the wave reads is on its way before anything is waited for
    h8_t b[NR][NT];
#pragma unroll
    for (int k = 0; k < NR; k++)
#pragma unroll
      for (int i = 0; i < NT; i++)
        b[k][i] = *reinterpret_cast<const h8_t*>(
            k_b + (int64_t(h) * c.rank + min(16 * (wv + 8 * k) + col, c.rank - 1)) * nope + min(32 * i + 8 * g, nope - 8));
    // (the parts of rows of no sequence are not used, nor made where all 16 are such)
    if (lo >= hi || t0 >= hi || t0 + 16 <= lo) return;
    const X* qr = q + min(max(t0 + col, lo), hi - 1) * q_stride + int64_t(h) * (nope + c.rope);
    float qv[NT][8];
#pragma unroll
    for (int i = 0; i < NT; i++) load8<X>(qr + min(32 * i + 8 * g, nope - 8), qv[i]);
    // the key part, its pair of the thread's token
    const int pairs = c.rope / 2, kt_ = tid / pairs, ki = tid % pairs;
    const bool key = kt_ < 16 && t0 + kt_ < c.n_tokens;
    const int key_t = min(max(t0 + min(kt_, 15), lo), hi - 1);
    const X* kp = q + key_t * q_stride + int64_t(h) * (nope + c.rope) + nope + 2 * ki;
    const float kx = float(kp[0]), ky = float(kp[1]);
    if (tid < 16) {
      s_key[tid] = 0;
      int first = t0 + tid, seq, pos;
      if (share > 1 && first < c.n_tokens && mla_locate_thread(c, first, seq, pos))
        first = mla_item_first(c, share, seq, first);
      s_first[tid] = first;
    }
    float ka = kx, kb = ky;
    if (rope.on) {
      int seq, pos;
      if (!mla_locate_thread(c, key_t, seq, pos)) pos = 0;
      const float2 cs = mla_cos_sin(rope, ki, pos);
      ka = kx * cs.x - ky * cs.y;
      kb = kx * cs.y + ky * cs.x;
    }
    if (!key) ka = kb = 0.f;
    // (f32: a token's values are brought near 1 by a power of two, so that their parts keep 22 bits whatever they are)
    int near = 0;
    if constexpr (sizeof(X) == 4) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) m = fmaxf(m, 32 * i + 8 * g < nope ? fabsf(qv[i][e]) : 0.f);
      m = max_over_groups(m);
      near = m > 0.f && m < INFINITY ? ilogbf(m) : 0;
    }
    h8_t ah[NT], al[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        _Float16 x, y;
        split2(32 * i + 8 * g < nope ? ldexpf(qv[i][e], -near) : 0.f, x, y);
        ah[i][e] = x, al[i][e] = y;
      }
    }
    int back[4];
#pragma unroll
    for (int e = 0; e < 4; e++) back[e] = sizeof(X) == 4 ? __shfl(near, 4 * g + e, kWave) : 0;
    f4_t v[NR];
    float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NR; k++) {
      const int r0 = 16 * (wv + 8 * k);
      f4_t hi = {0.f, 0.f, 0.f, 0.f}, lo = hi;
#pragma unroll
      for (int i = 0; i < NT; i++) {
        hi = mfma(ah[i], b[k][i], hi);
        if (sizeof(X) == 4) lo = mfma(al[i], b[k][i], lo);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[k][e] = r0 + col < c.rank ? ldexpf(hi[e] + lo[e], back[e]) : 0.f;
        mx[e] = fmaxf(mx[e], fabsf(v[k][e]));
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {  // over the 16 lanes of a row
      mx[e] = dpp_max<0xB1, 0xF>(mx[e]);
      mx[e] = dpp_max<0x4E, 0xF>(mx[e]);
      mx[e] = dpp_max<0x124, 0xF>(mx[e]);
      mx[e] = dpp_max<0x128, 0xF>(mx[e]);
      if (col == 0) s_max[wv][4 * g + e] = mx[e];
    }
    __syncthreads();
    if (key) atomicMax(&s_key[kt_], __float_as_uint(fmaxf(fabsf(ka), fabsf(kb))));
    __syncthreads();
    const int groups = (nh + 15) / 16;
    if (tid < 16) {  // the power of a token's largest value; 0 for a row of zeros, or one that is not finite
      float x = __uint_as_float(s_key[tid]);
#pragma unroll
      for (int w = 0; w < 8; w++) x = fmaxf(x, s_max[w][tid]);
      const int ex = x > 0.f && x < INFINITY ? ilogbf(x) : 0;
      s_ex[tid] = ex;
      if (t0 + tid < c.n_tokens)
        qa.factor[int64_t(s_first[tid]) * groups * 16 + (t0 + tid - s_first[tid]) * nh + h] = ldexpf(scale * 1.44269504088896341f, ex);
    }
    __syncthreads();
    // the parts by token and column in LDS, from there 16 bytes at a time
    constexpr int W = kMlaMaxRank + kMlaMaxRope + 8;
    constexpr bool TWO = sizeof(X) == 4;
    __shared__ __attribute__((aligned(16))) _Float16 s_part[TWO ? 2 : 1][16][W];
    auto put = [&](int t, int k, float x) {
      _Float16 hi, lo;
      split2(x, hi, lo);
      s_part[0][t][k] = hi;
      if (TWO) s_part[TWO][t][k] = lo;
    };
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int t = 4 * g + e, ex = s_ex[t];
#pragma unroll
      for (int k = 0; k < NR; k++) {
        const int r = 16 * (wv + 8 * k) + col;
        if (r < qa.rt) put(t, r, ldexpf(v[k][e], -ex));
      }
    }
    if (kt_ < 16) {
      const int ex = s_ex[kt_];
      put(kt_, qa.rt + 2 * ki, ldexpf(ka, -ex));
      put(kt_, qa.rt + 2 * ki + 1, ldexpf(kb, -ex));
    }
    const int cols = 32 * qa.kt, pad = cols - qa.rt - c.rope;  // columns of no pair
    for (int i = tid; i < 16 * pad; i += 512) put(i / pad, qa.rt + c.rope + i % pad, 0.f);
    __syncthreads();
    for (int i = tid; i < 16 * (cols / 8); i += 512) {
      const int t = i / (cols / 8), k = i % (cols / 8);  // 8 columns
      if (t0 + t >= c.n_tokens) break;
      const int first = s_first[t], row = (t0 + t - first) * nh + h;
      _Float16* p = qa.parts + ((int64_t(first) * groups + row / 16) * qa.kt + k / 4) * 512 + (k % 4) * 128 + (row % 16) * 8;
      *reinterpret_cast<h8_t*>(p) = *reinterpret_cast<const h8_t*>(&s_part[0][t][8 * k]);
      if (TWO) *reinterpret_cast<h8_t*>(p + qa.plane) = *reinterpret_cast<const h8_t*>(&s_part[TWO][t][8 * k]);
    }
    return;
  }
  // the plan: 512 tokens at a time, a scan of their units (the tiles, and for a token that has any as many as
  // beginning it takes)
  __shared__ int s_scan[8];
  int base = 0;
  for (int first = 0; first < c.n_tokens; first += 512) {
    const int t = first + tid;
    int seq = -1, pos = -1, end = 0, item = t;
    if (t < c.n_tokens) {
      if (mla_locate_thread(c, t, seq, pos)) {
        item = mla_item_first(c, share, seq, t);
        end = int(max(int64_t(0), min(int64_t(pos) + mla_item_tokens(c, share, seq, t), int64_t(c.max_len))));
      } else {
        seq = -1;
      }
    }
    const int mine = end > 0 && item == t ? (end + kMlaTile - 1) / kMlaTile + kMlaBegin : 0;
    int sum = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(sum, off, 64);
      if (lane >= off) sum += v;
    }
    if (lane == 63) s_scan[wv] = sum;
    __syncthreads();
    int before = base;
    for (int w = 0; w < 8; w++) {
      if (w < wv) before += s_scan[w];
      base += s_scan[w];
    }
    if (t < c.n_tokens) {
      plan.prefix[t] = before + sum - mine;
      plan.seq[t] = seq;
      plan.end[t] = end;
      plan.item[t] = item;
    }
    __syncthreads();
  }
  if (tid == 0) plan.prefix[c.n_tokens] = base;
}

// Units of a run: the plan's over the runs.
__device__ __forceinline__ int mla_per_run(int units, int runs) { return max((units + runs - 1) / runs, 1); }

// The last token whose prefix is not behind tile x, 64 candidates at a time.
__device__ __forceinline__ int mla_token_of(const int* prefix, int n, int x, int lane) {
  int lo = 0, len = n;  // the answer is in [lo, lo + len)
  while (len > 1) {
    const int step = (len + 63) / 64;
    const int i = lo + lane * step;
    const bool below = i < lo + len && prefix[i] <= x;
    const int k = max(__popcll(__ballot(below)) - 1, 0);
    const int at = lo + k * step;
    len = min(step, lo + len - at);
    lo = at;
  }
  return lo;
}

// Shape of the attend kernel: HG waves of 16 heads by KS waves of WR positions, RT + PT the padded widths,
// KV the cache's type.  LDS holds a step's rows in f16, the latents and then the key parts, so that neither 8
// rows' reads of one 16-byte chunk nor a transposing read's 32 bytes of 4 rows meet on a bank: rows of 1024
// bytes have 16 more after them (one address a lane for all reads), the chunks of shorter ones are swapped by the
// row's number.  An f16 cache is loaded straight into one of four such buffers; an f32 cache into a raw buffer,
// from which each wave turns its rows into a buffer of their upper and one of their lower parts.
template <int RT, int PT, int HG, int HW, int KS, typename KV>
struct AttendShape {
  static constexpr bool kWide = sizeof(KV) == 4;
  static constexpr int kWaves = HG * KS;
  static constexpr int kTile = kMlaTile;
  static constexpr int WR = kTile / KS;
  static constexpr int kRows = kTile / kWaves;  // rows a wave loads
  static constexpr bool kPad = RT == 512;
  static constexpr int kPitch = RT * 2 + (kPad ? 16 : 0);
  static constexpr int kLat = kTile * kPitch;
  static constexpr int kBuf = kLat + kTile * PT * 2;
  static constexpr int kBufs = kWide ? 2 : 4;
  static constexpr int kRaw = kWide ? kTile * (RT + PT) * 4 : 0;
  static constexpr int kMerge = KS > 1 ? HG * (KS - 1) * 16 * (RT + 4) * 4 : 0;  // over the buffers
  static constexpr int kLds = kBufs * kBuf + kRaw > kMerge ? kBufs * kBuf + kRaw : kMerge;
  // loads of 1024 bytes a wave issues for a step: of the latents, of the key parts
  static constexpr int kLoadsLat = kRows * RT * int(sizeof(KV)) / 1024;
  static constexpr int kLoadsKey = (kRows * PT * int(sizeof(KV)) + 1023) / 1024;
  static constexpr int kLoads = kLoadsLat + kLoadsKey;
  static_assert(kRows % 8 == 0 && kLds <= 160 * 1024, "tile shape");
  static_assert(HW == 1 || (KS == 1 && !kWide), "two 16s a wave have all positions of a step, and one part");
  __device__ static __forceinline__ constexpr int swap_lat(int r) { return kPad ? 0 : swap8(r); }
  __device__ static __forceinline__ constexpr int swap_key(int r) { return PT == 64 ? swap8(r) : swap4(r); }
  // byte of 16-byte chunk k (of the latent, or the key part) of row r
  __device__ static __forceinline__ int lat(int r, int k) { return r * kPitch + 16 * (k ^ swap_lat(r)); }
  __device__ static __forceinline__ int key(int r, int k) { return kLat + r * (PT * 2) + 16 * (k ^ swap_key(r)); }
};

// One run of tiles for HG x 16 heads.  Scores S^T[position][head] = K q'^T: A the cache rows from LDS, B
// the absorbed queries, held in registers for a token; the result has a head per lane column and positions
// 4g + e (g = lane / 16) of each 16, which is the B layout of the product O^T[r][head] += C^T p if 32 positions
// are taken in the order 4g .. 4g + 3, 16 + 4g .. 16 + 4g + 3: numerators never leave the lane, and C^T comes
// from the same LDS rows by transposing reads.  The accumulators (RT x 16 heads a wave) stay in registers;
// they are rescaled only where the maximum grew by more than 2^kAttendGrow.  With one part, the totals sum
// the numerators as the product rounds them.
//
// Registers allow one wave a SIMD, so a wave covers its own waits: a step's softmax runs between the products
// of the next step's scores, operands are read from LDS a group of products ahead, and the rows two steps on are
// on their way from the cache meanwhile (f16 cache; an f32 one has its LDS filled by the parts of one step).
//
// f16 activations: the queries and the numerators go in as one part.  An output is then off by 0.00038 of its size, of
// which its own rounding is 0.00021; 64 sequences of 128 heads take 122 us in all.  With queries of two parts (which
// leave no registers for two 16s of heads a wave) it is 0.00026 and 144 us, with numerators of two parts as well
// 0.00021 and 151; f32 activations are there for who needs them.
//
// HW 2 (f16 activations, more than 64 heads): two 16s of heads a wave, 128 a workgroup, so that each operand read
// from LDS serves two products, and cache rows go to one workgroup, not two; a step's softmax then stands between
// its products, as registers hold no second step's scores.  64 sequences of 100 to 4100 positions and 128 heads: 78 us
// against 86 with one 16 a wave; one of 131072 positions: 66 against 78 (and 4 to 5 us more in mla_values_kernel, as there
// are twice the partial rows).  With 64 heads (two waves sharing positions) it took 99 us and is not used.
//
// Measured (512 + 64 wide): one token of 131072 positions, 128 heads, f32 activations: 98 us, 740 TFLOP/s of two-part
// products; 32 sequences of 900 to 6000, 32 heads: 44 us, 2.9 TB/s.  Two-part products bound the first, the loads' and
// steps' latencies with one wave a SIMD the second; with f16 activations LDS reads (one 16 a wave: 2300 cycles a step
// of 32 positions, products 1090) and writing the partial rows (256 KB a workgroup of 128 heads, 14 us).
template <int RT, int PT, int HG, int HW, int KS, typename KV, bool TWO>
__global__ void __launch_bounds__(64 * HG * KS, 1)
    mla_attend_kernel(LatentCache c, MlaQueries qa, int nh, int share, MlaPlan plan, int runs,
                      float* __restrict__ part_o, float2* __restrict__ part_ml) {
  using S = AttendShape<RT, PT, HG, HW, KS, KV>;
  typedef uint32_t mask_t;  // a bit a position of a step
  constexpr mask_t ALL = ~mask_t(0);
  constexpr bool WIDE = S::kWide;
  constexpr int KT = (RT + PT) / 32, DT = RT / 16, RW = S::kRows, TR = S::kTile, WR = S::WR;
  constexpr int NT = WR / 16;  // 16-position tiles a wave
  __shared__ __attribute__((aligned(16))) uint8_t s_raw[S::kLds];
  const uint32_t lds0 = uint32_t(uintptr_t((lds_u8*)s_raw));

  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int hgw = wv % HG, kp = wv / HG;  // the wave's heads and positions
  // runs of the same tiles for different heads sit on one XCD (blocks go round the 8)
  const int rows_all = share * nh;  // of an item: its tokens' heads
  const int groups = (rows_all + 16 * HW * HG - 1) / (16 * HW * HG);
  const int b8 = blockIdx.x >> 3;
  const int run = (b8 / groups) * 8 + (blockIdx.x & 7), h0 = ((b8 % groups) * HG + hgw) * (16 * HW);
  const int n_tok = c.n_tokens;
  // the plan of up to 64 tokens from t0 on, a token a lane
  int t0 = 0;
  int w_prefix = plan.prefix[min(lane, n_tok)], w_seq = plan.seq[min(lane, n_tok - 1)], w_end = plan.end[min(lane, n_tok - 1)];
  const int tiles = plan.prefix[n_tok];
  const int per = mla_per_run(tiles, runs);
  int x = run * per;
  const int x_end = min(x + per, tiles);
  if (x >= x_end) return;

  auto window = [&](int t) {
    t0 = t;
    w_prefix = plan.prefix[min(t + lane, n_tok)];
    w_seq = plan.seq[min(t + lane, n_tok - 1)];
    w_end = plan.end[min(t + lane, n_tok - 1)];
  };
  int t = 0;
  if (n_tok > 63) {
    t = mla_token_of(plan.prefix, n_tok, x, lane);
    window(t);
  } else {
    t = __popcll(__ballot(lane < n_tok && w_prefix <= x)) - 1;
  }
  for (; x < x_end && t < n_tok; t++) {
    if (t - t0 > 62) window(t);
    const int first = __builtin_amdgcn_readlane(w_prefix, t - t0) + kMlaBegin;  // unit of the token's first tile
    const int last = min(__builtin_amdgcn_readlane(w_prefix, t - t0 + 1), x_end);
    x = max(x, first);
    if (last <= x) continue;  // a token without positions, or with none in this run
    const int seq = __builtin_amdgcn_readlane(w_seq, t - t0), end = __builtin_amdgcn_readlane(w_end, t - t0);
    const int32_t* table = c.table + seq * c.table_stride;
    const int p0 = (x - first) * TR, steps = last - x;
    const int rows_in = nh * mla_item_tokens(c, share, seq, t);
    int lim = end, top = end;  // positions that the lane's token attends to, and the item's first
    if (HW == 1 && share > 1) {
      const int64_t n = int64_t(c.lens[seq]) - c.starts[seq + 1] + t + 1;
      top = int(min(max(n, int64_t(0)), int64_t(end)));
      lim = int(min(max(n + min(h0 + col, rows_in - 1) / nh, int64_t(0)), int64_t(end)));
    }
    // of a step's rows that are there, those that the lane's token attends to
    auto seen = [&](mask_t here, int i) {
      if (HW > 1 || share == 1) return here;
      const int n = lim - (p0 + i * TR);
      return n >= TR ? here : n > 0 ? here & ((mask_t(1) << n) - 1) : mask_t(0);
    };

    // block ids of 64 blocks from block b0 on, a block a lane
    const int blocks = (end - 1) >> c.shift;  // the token's last
    int b0 = p0 >> c.shift;
    int ids = table[min(b0 + lane, blocks)];
    // where the rows of step i are (bytes, row r's in lane r; a row that is not there reads the pool's first
    // and is cleared once it has come), and which of them there are
    int64_t at = 0;
    auto find = [&](int i) {
      const int p = p0 + i * TR + (lane & (TR - 1));
      if ((min(p0 + i * TR + TR, end) - 1) >> c.shift >= b0 + 64) {
        b0 = (p0 + i * TR) >> c.shift;
        ids = table[min(b0 + lane, blocks)];
        asm volatile("" : "+v"(ids));  // waited for here, where it was loaded
      }
      const uint32_t blk = uint32_t(__shfl(ids, min((p >> c.shift) - b0, 63), kWave));
      const bool ok = p < end && blk < c.n_blocks;
      at = ok ? ((int64_t(blk) << c.shift) + (p & ((1 << c.shift) - 1))) * c.width * int(sizeof(KV)) : 0;
      return mask_t(__ballot(ok));
    };
    // load i of the wave's rows of that step, into buffer buf (or the raw rows)
    const uint8_t* const rows = static_cast<const uint8_t*>(c.rows);
    auto load = [&](int i, int buf) {
      constexpr int LB = RT * int(sizeof(KV)), KB = PT * int(sizeof(KV));  // bytes of a row's parts
      constexpr int NK = S::kLoadsKey;  // the key parts first: their addresses come through LDS
      const uint32_t dst = lds0 + (WIDE ? S::kBufs : buf) * S::kBuf;
      if (i < NK) {
        const int b = i * 1024 + 16 * lane, r = b / KB;
        const int64_t o = __shfl(at, min(wv * RW + r, TR - 1), kWave);
        const int sw = WIDE ? 0 : 16 * S::swap_key(r);
        const uint32_t to = dst + (WIDE ? TR * LB : S::kLat) + wv * RW * KB + i * 1024;
        if ((RW * KB) % 1024 == 0 || b < RW * KB)
          dma_lanes(rows + o + c.rank * int(sizeof(KV)) + min((b % KB) ^ sw, c.rope * int(sizeof(KV)) - 16), to);
      } else if constexpr (LB == 1024 && !WIDE) {
        const int r = wv * RW + i - NK;
        const uint32_t lo = __builtin_amdgcn_readlane(int(uint32_t(at)), r), hi = __builtin_amdgcn_readlane(int(at >> 32), r);
        dma_row(rows + ((int64_t(hi) << 32) | lo), min(16 * lane, 2 * c.rank - 16), dst + r * S::kPitch);
      } else {
        const int b = (i - NK) * 1024 + 16 * lane, r = b / LB;
        const int64_t o = __shfl(at, wv * RW + r, kWave);
        const int sw = WIDE ? 0 : 16 * S::swap_lat(r);
        dma_lanes(rows + o + min((b % LB) ^ sw, c.rank * int(sizeof(KV)) - 16), dst + wv * RW * LB + (i - NK) * 1024);
      }
    };
    // clears the wave's rows that are not there
    auto clear = [&](mask_t mask, int buf) {
      for (int r = wv * RW; r < wv * RW + RW; r++)
        if (!((mask >> r) & 1)) {
          uint8_t* p = s_raw + buf * S::kBuf;
          const u32x4 z = {0u, 0u, 0u, 0u};
          if (lane < RT / 8) *reinterpret_cast<u32x4*>(p + S::lat(r, lane)) = z;
          if (lane < PT / 8) *reinterpret_cast<u32x4*>(p + S::key(r, lane)) = z;
        }
    };
    // Rows that some of the item's tokens do not attend to: where the latent is not finite it is made zeros, as
    // those would take 0 * NaN from it, and the key part NaN for the others.
    auto scrub = [&](mask_t mask, int i, int buf) {
      if (HW > 1 || share == 1 || p0 + i * TR + TR <= top) return;
      for (int r = wv * RW; r < wv * RW + RW; r++) {
        if (!((mask >> r) & 1) || p0 + i * TR + r < top) continue;
        uint8_t* p = s_raw + buf * S::kBuf;
        bool odd = false;
        if (lane < RT / 8) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(p + S::lat(r, lane));
#pragma unroll
          for (int e = 0; e < 4; e++)
            odd |= (v[e] & 0x7C00u) == 0x7C00u || (v[e] & 0x7C000000u) == 0x7C000000u;
        }
        if (!__any(odd)) continue;
        const u32x4 z = {0u, 0u, 0u, 0u}, nan = {0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u};
        if (lane < RT / 8) *reinterpret_cast<u32x4*>(p + S::lat(r, lane)) = z;
        if (WIDE && lane < RT / 8) *reinterpret_cast<u32x4*>(p + S::kBuf + S::lat(r, lane)) = z;
        if (lane < PT / 8) *reinterpret_cast<u32x4*>(p + S::key(r, lane)) = nan;
      }
    };
    // an f32 cache: the wave's raw rows to their upper and lower parts
    auto convert = [&](mask_t mask) {
      auto part = [&](const uint8_t* src, int row, int dst) {
        const bool on = (mask >> row) & 1;
        float v[8];
        load8<float>(reinterpret_cast<const float*>(src), v);
        h8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          _Float16 a, b;
          split2(on ? v[e] : 0.f, a, b);
          hi[e] = a, lo[e] = b;
        }
        *reinterpret_cast<h8_t*>(s_raw + dst) = hi;
        *reinterpret_cast<h8_t*>(s_raw + S::kBuf + dst) = lo;
      };
      const uint8_t* raw = s_raw + S::kBufs * S::kBuf;
#pragma unroll 4
      for (int i = 0; i < RW * RT / 512; i++) {
        const int b = i * 64 + lane, r = wv * RW + b / (RT / 8), k = b % (RT / 8);
        part(raw + (r * RT + 8 * k) * 4, r, S::lat(r, k));
      }
      for (int b = lane; b < RW * PT / 8; b += 64) {
        const int r = wv * RW + b / (PT / 8), k = b % (PT / 8);
        part(raw + (TR * RT + r * PT + 8 * k) * 4, r, S::key(r, k));
      }
    };

    __syncthreads();  // the buffers are free of the token before
    constexpr int AHEAD = S::kBufs - 1;  // steps whose rows are on their way before the first
    mask_t mask[4] = {0, 0, 0, 0};     // which rows of the present step and the next three there are
#pragma unroll
    for (int j = 0; j < AHEAD; j++)
      if (j < steps) {
        mask[j] = find(j);
#pragma unroll
        for (int i = 0; i < S::kLoads; i++) load(i, j);
      }

    // the absorbed queries of the wave's heads
    h8_t qh[HW][KT], ql[TWO ? KT : 1];
    const int g16 = (nh + 15) / 16;
    float factor[HW];
#pragma unroll
    for (int w = 0; w < HW; w++) {
      const _Float16* const qp =
          qa.parts + (int64_t(t) * g16 + min(h0 / 16 + w, (rows_in + 15) / 16 - 1)) * KT * 512 + 8 * lane;
      // (columns past the item's rows hold what the workspace held: scores of 0 or NaN, which no maximum grows by)
      const int row = h0 + 16 * w + col;
      factor[w] = row < rows_in ? qa.factor[int64_t(t) * g16 * 16 + row] : 0.f;
#pragma unroll
      for (int i = 0; i < KT; i++) {
        qh[w][i] = *reinterpret_cast<const h8_t*>(qp + 512 * i);
        if constexpr (TWO) ql[i] = *reinterpret_cast<const h8_t*>(qp + qa.plane + 512 * i);
      }
    }
    f4_t o[HW][DT];
    float m[HW], l[HW];
#pragma unroll
    for (int w = 0; w < HW; w++) {
      m[w] = -INFINITY, l[w] = 0.f;
#pragma unroll
      for (int i = 0; i < DT; i++) o[w][i] = f4_t{0.f, 0.f, 0.f, 0.f};
    }

    // where the lane reads in a buffer, for each value of a chunk number's swapped bits; the rest is constant
    constexpr int NKL = S::kPad ? 1 : 2, NVV = S::kPad ? 1 : 4;
    int kl[NKL], kk[2], vv[NVV];
    {
      const int r = kp * WR + col;
#pragma unroll
      for (int i = 0; i < NKL; i++) kl[i] = S::lat(r, 4 * i + g);
      kk[0] = S::key(r, g), kk[1] = S::key(r, PT == 64 ? 4 + g : g);
      // lane l of a transposing read names 4 values of row 4g + col / 4 and gets column col of the 4 rows
      const int vr = kp * WR + 4 * g + (col >> 2);
#pragma unroll
      for (int d = 0; d < NVV; d++) vv[d] = S::lat(vr, 2 * d + ((col & 3) >> 1)) + 8 * (col & 1);
    }
    f4_t sa[NT], sb[NT];  // the scores of a step, in two sums
    constexpr int QN = KT;                             // groups of products: one k step each
    constexpr int KD = HW > 1 ? 2 : (NT == 1 ? 8 : 5) / (WIDE ? 2 : 1);  // groups whose operands are on their way
    h8_t ka[KD + 1][NT], kb[WIDE ? KD + 1 : 1][NT];
    auto read_k = [&](int k, const uint8_t* kv) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const uint8_t* p = kv + (k < RT / 32 ? kl[k % NKL] + 64 * (k - k % NKL) + 16 * j * S::kPitch
                                             : kk[(k - RT / 32) & 1] + 16 * j * PT * 2);
        ka[k % (KD + 1)][j] = *reinterpret_cast<const h8_t*>(p);
        if constexpr (WIDE) kb[k % (KD + 1)][j] = *reinterpret_cast<const h8_t*>(p + S::kBuf);
      }
    };
    // the scores of the step in buffer kv; between the groups of products, between(group)
    auto scores = [&](const uint8_t* kv, f4_t (&a)[NT], f4_t (&b)[NT], auto between) {
#pragma unroll
      for (int j = 0; j < NT; j++) a[j] = b[j] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KD && k < QN; k++) read_k(k, kv);
#pragma unroll
      for (int k = 0; k < QN; k++) {
        if (k + KD < QN) read_k(k + KD, kv);
        between(k);
        constexpr int M = KD + 1;
#pragma unroll
        for (int j = 0; j < NT; j++) {
          if (!TWO && (k & 1)) b[j] = mfma(ka[k % M][j], qh[0][k], b[j]);  // two chains
          else a[j] = mfma(ka[k % M][j], qh[0][k], a[j]);
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
          if constexpr (TWO) b[j] = mfma(ka[k % M][j], ql[k], b[j]);
          if constexpr (WIDE) b[j] = mfma(kb[k % M][j], qh[0][k], b[j]);
        }
        if (k % 3 == 2) __builtin_amdgcn_sched_barrier(0);  // reads stay ahead, and no further
      }
    };
    // the softmax of a step's scores, in 16 pieces to go between products: each result is pinned where it is
    // made (the compiler would move it to its use)
    constexpr int PIECES = 16, NS = 4 * NT;
    float sc[NS], mx = 0.f, ref = 0.f, alpha = 1.f, sum = 0.f;
    bool grew = false;
    _Float16 ph[NS], pl[NS];
    auto soft = [&](int piece, mask_t here) {
      if (piece < 4) {
        const uint32_t own = uint32_t(here >> (kp * WR)) >> (4 * g);  // bit 16 j + e: position 4g + e of tile j
#pragma unroll
        for (int n = piece * NS / 4; n < (piece + 1) * NS / 4; n++) {
          const int j = n / 4, e = n % 4;
          const float s = (sa[j][e] + sb[j][e]) * factor[0];
          sc[n] = own & (1u << (16 * j + e)) ? s : -INFINITY;
          asm volatile("" : "+v"(sc[n]));
        }
      } else if (piece == 4) {
        mx = sc[0];
#pragma unroll
        for (int n = 1; n < NS; n++) mx = fmaxf(mx, sc[n]);
        asm volatile("" : "+v"(mx));
      } else if (piece == 5) {
        mx = max_over_groups(mx);
        asm volatile("" : "+v"(mx));
      } else if (piece == 6) {
        grew = __any(mx > m[0] + kAttendGrow);
        const float mn = grew ? fmaxf(m[0], mx) : m[0];
        ref = mn == -INFINITY ? 0.f : mn;
        alpha = __builtin_amdgcn_exp2f(m[0] - ref);  // 0 at first: exp2(-inf)
        ref -= kAttendLift;
        m[0] = mn;
        l[0] *= alpha;
        asm volatile("" : "+v"(ref), "+v"(alpha), "+v"(m[0]), "+v"(l[0]));
      } else if (piece < 15) {
#pragma unroll
        for (int n = (piece - 7) * NS / 8; n < (piece - 6) * NS / 8; n++) {
          const float p = __builtin_amdgcn_exp2f(sc[n] - ref);
          split2(p, ph[n], pl[n]);
          sc[n] = TWO ? p : float(ph[n]);
          asm volatile("" : "+v"(sc[n]));
        }
      } else {
        sum = sc[0];
#pragma unroll
        for (int n = 1; n < NS; n++) sum += sc[n];
        l[0] += sum;
      }
    };
    // O^T += C^T p from buffer kv
    auto values = [&](const uint8_t* kv) {
      if (grew) {
#pragma unroll
        for (int d = 0; d < DT; d++) {
          asm volatile("" : "+a"(o[0][d]));  // in accumulation registers up to here: else all are copied every step
          o[0][d] *= alpha;
        }
      }
      auto tr = [&](int d, int j, int plane) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s4*)(kv + vv[d % NVV] + plane * S::kBuf + 32 * (d - d % NVV) + 16 * j * S::kPitch));
      };
      constexpr int VG = 2, VN = DT / VG;               // tiles of 16 latent columns a group
      constexpr int VD = (NT == 1 ? 6 : 3) / (WIDE ? 2 : 1);  // groups on their way
      typedef std::conditional_t<NT == 1, h4_t, h8_t> v_t;
      v_t bh, bl, va[VD + 1][VG], vl[WIDE ? VD + 1 : 1][VG];
#pragma unroll
      for (int e = 0; e < 4 * NT; e++) bh[e] = ph[e], bl[e] = pl[e];
      auto operand = [&](int d, int plane) {
        if constexpr (NT == 1) return __builtin_bit_cast(h4_t, tr(d, 0, plane));
        else
          return __builtin_bit_cast(h8_t,
                                    __builtin_shufflevector(tr(d, 0, plane), tr(d, 1, plane), 0, 1, 2, 3, 4, 5, 6, 7));
      };
      auto read_v = [&](int grp) {
#pragma unroll
        for (int i = 0; i < VG; i++) {
          va[grp % (VD + 1)][i] = operand(grp * VG + i, 0);
          if constexpr (WIDE) vl[grp % (VD + 1)][i] = operand(grp * VG + i, 1);
        }
      };
      auto add = [&](f4_t& d, v_t v, v_t p) {
        if constexpr (NT == 1) d = __builtin_amdgcn_mfma_f32_16x16x16f16(v, p, d, 0, 0, 0);
        else d = mfma(v, p, d);
      };
#pragma unroll
      for (int grp = 0; grp < VD && grp < VN; grp++) read_v(grp);
#pragma unroll
      for (int grp = 0; grp < VN; grp++) {
        if (grp + VD < VN) read_v(grp + VD);
        constexpr int M = VD + 1;
#pragma unroll
        for (int i = 0; i < VG; i++) add(o[0][grp * VG + i], va[grp % M][i], bh);
        if constexpr (TWO)
#pragma unroll
          for (int i = 0; i < VG; i++) add(o[0][grp * VG + i], va[grp % M][i], bl);
        if constexpr (WIDE)
#pragma unroll
          for (int i = 0; i < VG; i++) add(o[0][grp * VG + i], vl[grp % M][i], bh);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    if constexpr (HW > 1) {
      // Two 16s of heads a wave, each operand read from LDS for both: products bound a step, not LDS, and the
      // softmax stands between them (registers hold no second step's scores)
      static_assert(!TWO && NT == 2);
      for (int i = 0; i < steps; i++) {
        if (AHEAD > 1 && i + AHEAD <= steps) dma_wait<(AHEAD - 1) * S::kLoads>();
        else dma_wait<0>();
        const mask_t here = mask[0];
        if (here != ALL) clear(here, i % S::kBufs);
        __syncthreads();  // the step's rows are there, and the step before has been read
        if (i + AHEAD < steps) {
          mask[AHEAD] = find(i + AHEAD);
#pragma unroll
          for (int n = 0; n < S::kLoads; n++) load(n, (i + AHEAD) % S::kBufs);
        }
        const uint8_t* const kv = s_raw + (i % S::kBufs) * S::kBuf;
        f4_t sx[HW][NT];
#pragma unroll
        for (int w = 0; w < HW; w++)
#pragma unroll
          for (int j = 0; j < NT; j++) sx[w][j] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KD && k < QN; k++) read_k(k, kv);
#pragma unroll
        for (int k = 0; k < QN; k++) {
          if (k + KD < QN) read_k(k + KD, kv);
#pragma unroll
          for (int w = 0; w < HW; w++)
#pragma unroll
            for (int j = 0; j < NT; j++) sx[w][j] = mfma(ka[k % (KD + 1)][j], qh[w][k], sx[w][j]);
          if (k % 2) __builtin_amdgcn_sched_barrier(0);
        }
        h8_t p[HW];
        float by[HW];
        bool grown = false;
        const uint32_t own = uint32_t(here >> (kp * WR)) >> (4 * g);
#pragma unroll
        for (int w = 0; w < HW; w++) {
          float x8[8], top = -INFINITY;
#pragma unroll
          for (int n = 0; n < 8; n++) {
            x8[n] = own & (1u << (16 * (n / 4) + n % 4)) ? sx[w][n / 4][n % 4] * factor[w] : -INFINITY;
            top = fmaxf(top, x8[n]);
          }
          top = max_over_groups(top);
          const bool up = __any(top > m[w] + kAttendGrow);
          const float mn = up ? fmaxf(m[w], top) : m[w];
          const float at0 = mn == -INFINITY ? 0.f : mn;
          by[w] = __builtin_amdgcn_exp2f(m[w] - at0);
          m[w] = mn;
          grown |= up;
          float add8 = 0.f;
#pragma unroll
          for (int n = 0; n < 8; n++) {
            p[w][n] = _Float16(__builtin_amdgcn_exp2f(x8[n] - (at0 - kAttendLift)));
            add8 += float(p[w][n]);
          }
          l[w] = l[w] * by[w] + add8;
        }
        if (grown) {
#pragma unroll
          for (int w = 0; w < HW; w++)
#pragma unroll
            for (int d = 0; d < DT; d++) {
              asm volatile("" : "+a"(o[w][d]));
              o[w][d] *= by[w];
              asm volatile("" : "+a"(o[w][d]));
            }
        }
        auto operand = [&](int d) {
          auto tr = [&](int j) {
            return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s4*)(kv + vv[d % NVV] + 32 * (d - d % NVV) + 16 * j * S::kPitch));
          };
          return __builtin_bit_cast(h8_t, __builtin_shufflevector(tr(0), tr(1), 0, 1, 2, 3, 4, 5, 6, 7));
        };
        constexpr int VD = 4;  // operands on their way
        h8_t va[VD + 1];
#pragma unroll
        for (int d = 0; d < VD; d++) va[d] = operand(d);
#pragma unroll
        for (int d = 0; d < DT; d++) {
          if (d + VD < DT) va[(d + VD) % (VD + 1)] = operand(d + VD);
#pragma unroll
          for (int w = 0; w < HW; w++) o[w][d] = mfma(va[d % (VD + 1)], p[w], o[w][d]);
          if (d % 2) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < AHEAD; n++) mask[n] = mask[n + 1];
      }
    } else if constexpr (WIDE) {
      for (int i = 0; i < steps; i++) {
        dma_wait<0>();
        __syncthreads();  // the parts of the step before have been read
        const mask_t here = mask[0];
        convert(here);
        scrub(here, i, 0);
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the raw rows have been read
        const bool more = i + 1 < steps;
        if (more) {
          mask[0] = find(i + 1);
#pragma unroll
          for (int n = 0; n < S::kLoadsKey; n++) load(n, 0);
        }
        __syncthreads();
        scores(s_raw, sa, sb, [&](int grp) {
          if (more)  // the next step's loads, a few a group
#pragma unroll
            for (int n = grp * S::kLoadsLat / QN; n < (grp + 1) * S::kLoadsLat / QN; n++) load(S::kLoadsKey + n, 0);
        });
#pragma unroll
        for (int n = 0; n < PIECES; n++) soft(n, seen(here, i));
        values(s_raw);
      }
    } else {
      // step i: its scores are there; the next step's rows have come, those of two more are on their way
      if (steps > 2) dma_wait<2 * S::kLoads>();
      else if (steps > 1) dma_wait<S::kLoads>();
      else dma_wait<0>();
      if (mask[0] != ALL) clear(mask[0], 0);
      scrub(mask[0], 0, 0);
      __syncthreads();
      scores(s_raw, sa, sb, [](int) {});
      for (int i = 0; i < steps; i++) {
        // (after the last step the scores are those of some rows still in LDS, and not used: a second copy of
        // the products for it would cost their registers)
        const int nb = (i + 1) & 3, fb = (i + 3) & 3;
        const bool more = i + 3 < steps;
        if (i + 2 < steps) dma_wait<S::kLoads>();
        else dma_wait<0>();
        if (i + 1 < steps && mask[1] != ALL) clear(mask[1], nb);
        if (i + 1 < steps) scrub(mask[1], i + 1, nb);
        __syncthreads();  // the next step's rows are there, and the step before has been read
        if (more) {
          mask[3] = find(i + 3);
#pragma unroll
          for (int n = 0; n < S::kLoads; n++) load(n, fb);
        }
        const mask_t here = seen(mask[0], i);
        f4_t na[NT], nb2[NT];
        scores(s_raw + nb * S::kBuf, na, nb2, [&](int grp) {
#pragma unroll
          for (int n = grp * PIECES / QN; n < (grp + 1) * PIECES / QN; n++) soft(n, here);
        });
        values(s_raw + (i & 3) * S::kBuf);
#pragma unroll
        for (int j = 0; j < NT; j++) sa[j] = na[j], sb[j] = nb2[j];
        mask[0] = mask[1], mask[1] = mask[2], mask[2] = mask[3];
      }
    }
#pragma unroll
    for (int w = 0; w < HW; w++) l[w] = sum_over_groups(l[w]);

    // waves of the same heads merge through LDS, over the buffers
    const int64_t slot = run + mla_item(share, seq, t);
    if constexpr (KS > 1) {
      static_assert(KS == 2);
      constexpr int W = RT + 4;
      float* const at = reinterpret_cast<float*>(s_raw) + hgw * 16 * W + col * W;
      __syncthreads();
      if (kp) {
#pragma unroll
        for (int d = 0; d < DT; d++) *reinterpret_cast<f4_t*>(at + 16 * d + 4 * g) = o[0][d];
        if (g == 0) at[RT] = m[0], at[RT + 1] = l[0];
      }
      __syncthreads();
      if (kp == 0) {
        const float mt = fmaxf(m[0], at[RT]), top = mt == -INFINITY ? 0.f : mt;
        const float a = __builtin_amdgcn_exp2f(m[0] - top), b = __builtin_amdgcn_exp2f(at[RT] - top);
        l[0] = a * l[0] + b * at[RT + 1];
#pragma unroll
        for (int d = 0; d < DT; d++) o[0][d] = a * o[0][d] + b * *reinterpret_cast<const f4_t*>(at + 16 * d + 4 * g);
        m[0] = mt;
      }
    }
#pragma unroll
    for (int w = 0; w < HW; w++) {
      const int head = h0 + 16 * w + col;
      if (kp || head >= rows_in) continue;
      float* po = part_o + (slot * rows_all + head) * c.rank;
#pragma unroll
      for (int d = 0; d < DT; d++)
        if (16 * d + 4 * g < c.rank) *reinterpret_cast<f4_t*>(po + 16 * d + 4 * g) = o[w][d];
      if (g == 0) part_ml[slot * rows_all + head] = make_float2(m[w], l[w]);
    }
    x = last;
  }
}

// out[t][h] = W_uv[h] o[t][h], o the merged partials: a block of 8 waves per head and up to TB tokens.  The
// weights' rows (16 of them a wave, its MFMA operand) are on their way while the partials are merged, by 8 / TB
// waves a token (TB 16: a wave, two tokens), into LDS.  Bound by the partials' bytes and, for a token, latency: one
// token of 128 heads and 128 runs (33 MB of partials) 12 us, 64 tokens with 256 runs (84 MB) 26 us, 3.2 TB/s.
template <typename X, int RT, int TB>
__global__ void __launch_bounds__(512) mla_values_kernel(LatentCache c, int nh, const float* __restrict__ part_o,
                                                         const float2* __restrict__ part_ml, MlaPlan plan, int runs,
                                                         int share,
                                                         const _Float16* __restrict__ v_b, int v_dim, X* __restrict__ out, int64_t out_stride) {
  constexpr int KT = RT / 32, P = RT + 8, NW = 8, U = 4, WPT = TB < 8 ? 8 / TB : 1;
  __shared__ __attribute__((aligned(16))) _Float16 s_hi[16][P], s_lo[16][P];
  __shared__ __attribute__((aligned(16))) float s_acc[WPT > 1 ? NW : 1][RT];
  __shared__ float s_m[NW], s_l[NW];
  int h, t0;
  if (!mla_head_block(blockIdx.x, nh, (c.n_tokens + TB - 1) / TB, h, t0)) return;
  t0 *= TB;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int g = lane >> 4, col = lane & 15;
  const int vt = (v_dim + 15) / 16;
  h8_t b[KT];
  auto weights = [&](int tile) {
    const _Float16* w = v_b + (int64_t(h) * v_dim + min(16 * tile + col, v_dim - 1)) * c.rank;
#pragma unroll
    for (int i = 0; i < KT; i++) b[i] = *reinterpret_cast<const h8_t*>(w + min(32 * i + 8 * g, c.rank - 8));
  };
  weights(min(wv, vt - 1));
  const int per = mla_per_run(plan.prefix[c.n_tokens], runs);
  const int r0 = min(8 * lane, c.rank - 8);

  // partials w0, w0 + by, ... below w1 of row `row` of item `item`, of which lane l holds elements 8l ..: sum,
  // maximum, total
  float acc[8], m, l;
  auto merge = [&](int item, int row, int w0, int w1, int by) {
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = 0.f;
    m = -INFINITY, l = 0.f;
    for (int w = w0; w < w1; w += by * U) {
      float4 lo[U], hi[U];
      float2 ml[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t at = int64_t(min(w + u * by, w1 - 1) + item) * (share * nh) + row;
        const float* p = part_o + at * c.rank + r0;
        lo[u] = *reinterpret_cast<const float4*>(p);
        hi[u] = *reinterpret_cast<const float4*>(p + 4);
        ml[u] = part_ml[at];
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; u++)
        if (w + u * by < w1) mn = fmaxf(mn, ml[u].x);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float a = __builtin_amdgcn_exp2f(m - ref);
      l *= a;
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] *= a;
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (w + u * by >= w1) continue;
        const float f = __builtin_amdgcn_exp2f(ml[u].x - ref);
        l += f * ml[u].y;
        acc[0] += f * lo[u].x, acc[1] += f * lo[u].y, acc[2] += f * lo[u].z, acc[3] += f * lo[u].w;
        acc[4] += f * hi[u].x, acc[5] += f * hi[u].y, acc[6] += f * hi[u].z, acc[7] += f * hi[u].w;
      }
      m = mn;
    }
  };
  auto keep = [&](int row, float total) {
    const float inv = total != 0.f ? 1.0f / total : 0.f;
    if (8 * lane < RT) {
      h8_t hi, lo;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        _Float16 x, y;
        split2(8 * lane < c.rank ? acc[e] * inv : 0.f, x, y);
        hi[e] = x, lo[e] = y;
      }
      *reinterpret_cast<h8_t*>(&s_hi[row][8 * lane]) = hi;
      *reinterpret_cast<h8_t*>(&s_lo[row][8 * lane]) = lo;
    }
  };
#pragma unroll
  for (int i = wv / WPT; i < TB; i += NW / WPT) {
    const int t = t0 + i;
    int w0 = 0, w1 = 0, first = t, item = t;
    if (t < c.n_tokens) {
      if (share > 1) first = plan.item[t], item = mla_item(share, plan.seq[t], first);
      const int a = plan.prefix[first] + kMlaBegin, e = plan.prefix[first + 1];
      w0 = a / per;
      w1 = e > a ? (e - 1) / per + 1 : w0;
    }
    merge(item, (t - first) * nh + h, w0 + wv % WPT, w1, WPT);
    if constexpr (WPT == 1) keep(i, l);
  }
  if constexpr (WPT > 1) {
    if (8 * lane < RT) {
      reinterpret_cast<float4*>(&s_acc[wv][8 * lane])[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      reinterpret_cast<float4*>(&s_acc[wv][8 * lane])[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
    if (lane == 0) s_m[wv] = m, s_l[wv] = l;
    __syncthreads();
    if (wv < TB) {
      float mt = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < WPT; w++) mt = fmaxf(mt, s_m[wv * WPT + w]);
      const float ref = mt == -INFINITY ? 0.f : mt;
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] = 0.f;
#pragma unroll
      for (int w = 0; w < WPT; w++) {
        const float f = __builtin_amdgcn_exp2f(s_m[wv * WPT + w] - ref);
        total += f * s_l[wv * WPT + w];
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] += f * s_acc[wv * WPT + w][min(8 * lane, RT - 8) + e];
      }
      keep(wv, total);
    }
  }
  __syncthreads();
  // (rows from TB on of the product's 16 are those of other tokens, and not stored)
  const int row = col & (TB - 1);
  for (int tile = wv; tile < vt; tile += NW) {
    if (tile != wv) weights(tile);
    f4_t hi = {0.f, 0.f, 0.f, 0.f}, lo = hi;
#pragma unroll
    for (int i = 0; i < KT; i++) {
      hi = mfma(*reinterpret_cast<const h8_t*>(&s_hi[row][32 * i + 8 * g]), b[i], hi);
      lo = mfma(*reinterpret_cast<const h8_t*>(&s_lo[row][32 * i + 8 * g]), b[i], lo);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = 4 * g + e, t = t0 + i, v = 16 * tile + col;
      if (i < TB && t < c.n_tokens && v < v_dim && plan.seq[t] >= 0)
        out[t * out_stride + int64_t(h) * v_dim + v] = X(hi[e] + lo[e]);
    }
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
  if (n_tokens > (1 << 19) || c->n_seqs > (1 << 19) || c->n_blocks > INT32_MAX)
    return fail(JERO_ERR_TENSOR_BOUNDS, w + "more than 2^19 tokens or sequences, or 2^31 - 1 blocks");
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
  // (a model's calls all ask for the same: 32 powers cost the host a launch's time)
  static thread_local struct {
    float theta = 0.f;
    int dim = 0;
    MlaRope rope{};
  } last;
  if (last.theta != theta || last.dim != rope_dim) {
    last.theta = theta;
    last.dim = rope_dim;
    last.rope.on = 1;
    for (int i = 0; i < rope_dim / 2; i++)
      last.rope.turns[i] = std::pow(double(theta), -2.0 * i / rope_dim) / 6.283185307179586476925;
  }
  *out = last.rope;
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
  if (vec)                                                                                                          \
    hipLaunchKernelGGL((mla_append_kernel<X, KV, true>), grid, dim3(256), 0, s, c, static_cast<const X*>(x_dev),   \
                       x_stride, norm_dev, eps, rope);                                                              \
  else                                                                                                              \
    hipLaunchKernelGGL((mla_append_kernel<X, KV, false>), grid, dim3(256), 0, s, c, static_cast<const X*>(x_dev),  \
                       x_stride, norm_dev, eps, rope)
  const int size = act_dtype == JERO_F32 ? 4 : 2;
  const bool vec = !((reinterpret_cast<uintptr_t>(x_dev) | uintptr_t(x_stride * size)) & 15u);
  if (act_dtype == JERO_F32) {
    if (f16) {
      JERO_APPEND(float, _Float16);
    } else {
      JERO_APPEND(float, float);
    }
  } else if (f16) {
    JERO_APPEND(_Float16, _Float16);
  } else {
    JERO_APPEND(_Float16, float);
  }
#undef JERO_APPEND
  return check_launch("mla_append");
}

namespace jero {

// Where the parts of the absorbed form's workspace are.
struct AbsorbedSpace {
  size_t factor, part_o, part_ml, plan, bytes;
  int rt, pt;  // padded widths: the smallest that the attend kernel is built for
};

// Tokens an item: as many as sequences have on average, and 64 rows of heads hold.  Only n_tokens and n_seqs are
// known here: where most sequences have one token, each is by itself.  Measured, attend and value product, tokens by
// themselves and together: 7 sequences x 2-4 tokens, 20 heads, 40-2500 positions of f32 31 + 10 and 24 + 12 us; 16
// sequences of 2000-6000, 32 heads 126 + 17 and 88 + 20; 16 heads, f16 53 + 10 and 37 + 12.
static int absorbed_share(const jero_latent_cache* c, int64_t n_tokens, int n_heads) {
  if (!c->starts_dev || n_tokens <= c->n_seqs || n_heads > 32) return 1;
  return int(std::min<int64_t>(64 / n_heads, (n_tokens + c->n_seqs - 1) / c->n_seqs));
}

static AbsorbedSpace absorbed_space(const jero_latent_cache* c, int64_t n_tokens, int n_heads) {
  auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  const int share = absorbed_share(c, n_tokens, n_heads);
  const size_t items = size_t(share > 1 ? n_tokens / share + c->n_seqs : n_tokens);
  const size_t parts = (items + kMlaRuns) * share * n_heads;
  const size_t rows16 = size_t(n_tokens) * ((n_heads + 15) / 16 * 16);
  AbsorbedSpace s;
  s.rt = c->rank <= 128 && c->rope_dim <= 32 ? 128 : c->rank <= 256 ? 256 : 512;
  s.pt = s.rt == 128 ? 32 : 64;
  s.factor = up(rows16 * (s.rt + s.pt) * 4);
  s.part_o = s.factor + up(rows16 * 4);
  s.part_ml = s.part_o + up(parts * c->rank * 4);
  s.plan = s.part_ml + up(parts * 8);
  s.bytes = s.plan + up((4 * size_t(n_tokens) + 1) * 4);
  return s;
}

template <int RT, int PT, int HG, int HW, int KS, typename KV, bool TWO>
static void launch_attend(const LatentCache& c, const MlaQueries& qa, int nh, int share, const MlaPlan& plan, int runs,
                          float* part_o, float2* part_ml, hipStream_t s) {
  const int groups = (share * nh + 16 * HW * HG - 1) / (16 * HW * HG);
  hipLaunchKernelGGL((mla_attend_kernel<RT, PT, HG, HW, KS, KV, TWO>), dim3(unsigned(runs) * groups), dim3(64 * HG * KS),
                     0, s, c, qa, nh, share, plan, runs, part_o, part_ml);
}

// Heads a workgroup: 16 by each of its 1, 2 or 4 waves' worth; with fewer than 4 others share the positions.
// f16 activations, whose queries are one part, leave the registers for two 16s a wave from 65 heads on.
static int attend_heads(int nh, bool one_part) { return nh <= 16 ? 16 : nh <= 32 ? 32 : nh <= 64 || !one_part ? 64 : 128; }

template <int RT, int PT, typename KV, bool TWO>
static void launch_attend_heads(const LatentCache& c, const MlaQueries& qa, int nh, int share, const MlaPlan& plan, int runs,
                                float* part_o, float2* part_ml, hipStream_t s) {
  const int heads = attend_heads(share * nh, !TWO);
  if (heads == 16) launch_attend<RT, PT, 1, 1, 2, KV, TWO>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
  else if (heads == 32) launch_attend<RT, PT, 2, 1, 2, KV, TWO>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
  else if (heads == 64) launch_attend<RT, PT, 4, 1, 1, KV, TWO>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
  else if constexpr (!TWO) launch_attend<RT, PT, 4, 2, 1, KV, TWO>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
}

template <int RT, int PT>
static void launch_attend_types(bool f32_act, bool f32_kv, const LatentCache& c, const MlaQueries& qa, int nh,
                                int share, const MlaPlan& plan, int runs, float* part_o, float2* part_ml, hipStream_t s) {
  if (f32_kv) launch_attend_heads<RT, PT, float, true>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
  else if (f32_act) launch_attend_heads<RT, PT, _Float16, true>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
  else launch_attend_heads<RT, PT, _Float16, false>(c, qa, nh, share, plan, runs, part_o, part_ml, s);
}

}  // namespace jero

extern "C" size_t jero_hip_mla_absorbed_workspace_bytes(const jero_latent_cache* cache, int64_t n_tokens, int n_heads) {
  if (!cache || n_tokens < 1 || n_heads < 1 || cache->rank < 1 || cache->rope_dim < 1 || cache->n_seqs < 1) return 0;
  return absorbed_space(cache, n_tokens, n_heads).bytes;
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
  // the plan's units (32 positions, and 4 a token more at most) and the grids' work items are 32-bit
  if (n_tokens * cache->max_len > (int64_t(1) << 34) || n_tokens * n_heads > (int64_t(1) << 25))
    return fail(JERO_ERR_CAPABILITY_MISMATCH, "mla_absorbed_attention: more than 2^34 tokens x max_len or 2^25 tokens x heads");
  const AbsorbedSpace sp = absorbed_space(cache, n_tokens, n_heads);
  void* ws = workspace_dev;
  if ((rc = absorbed_workspace(sp.bytes, &ws, workspace_bytes, kName))) return rc;
  const LatentCache c = mla_cache_of(cache, n_tokens);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* const w = static_cast<uint8_t*>(ws);
  MlaQueries qa;
  qa.parts = reinterpret_cast<_Float16*>(w);
  qa.factor = reinterpret_cast<float*>(w + sp.factor);
  qa.plane = n_tokens * ((n_heads + 15) / 16 * 16) * (sp.rt + sp.pt);
  qa.rt = sp.rt;
  qa.kt = (sp.rt + sp.pt) / 32;
  float* part_o = reinterpret_cast<float*>(w + sp.part_o);
  float2* part_ml = reinterpret_cast<float2*>(w + sp.part_ml);
  MlaPlan plan;
  plan.prefix = reinterpret_cast<int*>(w + sp.plan);
  plan.seq = plan.prefix + n_tokens + 1;
  plan.end = plan.seq + n_tokens;
  plan.item = plan.end + n_tokens;
  const _Float16 *kb = static_cast<const _Float16*>(k_b_dev), *vb = static_cast<const _Float16*>(v_b_dev);
  const bool f32 = act_dtype == JERO_F32;
  const int share = absorbed_share(cache, n_tokens, n_heads);
  const int heads = attend_heads(share * n_heads, !f32), groups = (share * n_heads + heads - 1) / heads;
  const int runs = kMlaRuns / groups / 8 * 8;  // (groups: 16 at most)

  const dim3 ga(mla_head8_blocks(n_heads, int((n_tokens + 15) / 16)) + 1);
#define JERO_ABSORB(X, NT)                                                                                         \
  hipLaunchKernelGGL((mla_absorb_kernel<X, NT>), ga, dim3(512), 0, s, c, static_cast<const X*>(q_dev), q_stride, n_heads, \
                     nope_dim, kb, rope, scale, qa, plan, share)
  if (nope_dim <= 128) {
    if (f32) JERO_ABSORB(float, 4);
    else JERO_ABSORB(_Float16, 4);
  } else {
    if (f32) JERO_ABSORB(float, 8);
    else JERO_ABSORB(_Float16, 8);
  }
#undef JERO_ABSORB
  if ((rc = check_launch("mla absorb"))) return rc;

  const bool wide = cache->kv_dtype == JERO_KV_F32;
  if (sp.rt == 128)
    launch_attend_types<128, 32>(f32, wide, c, qa, n_heads, share, plan, runs, part_o, part_ml, s);
  else if (sp.rt == 256)
    launch_attend_types<256, 64>(f32, wide, c, qa, n_heads, share, plan, runs, part_o, part_ml, s);
  else
    launch_attend_types<512, 64>(f32, wide, c, qa, n_heads, share, plan, runs, part_o, part_ml, s);
  if ((rc = check_launch("mla attend"))) return rc;

  // tokens a block: as many as leave 64 blocks or more, so that the weights are read seldom (21 tokens of 20 heads:
  // by 1 14.1 us, by 4 10.5, by 16 16.4; 32 of 32: 26.6, 10.9, 14.3; 16 of 128: 57, 24, 20.6; 64 of 128: 187, 64, 27)
  const int64_t rows = n_tokens * n_heads;
#define JERO_VALUES_TB(X, RT, TB)                                                                                    \
  hipLaunchKernelGGL((mla_values_kernel<X, RT, TB>), dim3(mla_head_blocks(n_heads, int((n_tokens + TB - 1) / TB))), \
                     dim3(512), 0, s, c, n_heads, part_o, part_ml, plan, runs, share, vb, v_dim,                           \
                     static_cast<X*>(out_dev), out_stride)
#define JERO_VALUES(X, RT)                                                                                       \
  if (n_tokens < 2 || rows < 256) JERO_VALUES_TB(X, RT, 1);                                                      \
  else if (rows < 2048) JERO_VALUES_TB(X, RT, 4);                                                                \
  else JERO_VALUES_TB(X, RT, 16)
  if (sp.rt == 128) {
    if (f32) {
      JERO_VALUES(float, 128);
    } else {
      JERO_VALUES(_Float16, 128);
    }
  } else if (sp.rt == 256) {
    if (f32) {
      JERO_VALUES(float, 256);
    } else {
      JERO_VALUES(_Float16, 256);
    }
  } else if (f32) {
    JERO_VALUES(float, 512);
  } else {
    JERO_VALUES(_Float16, 512);
  }
#undef JERO_VALUES_TB
#undef JERO_VALUES
  return check_launch("mla values");
}
