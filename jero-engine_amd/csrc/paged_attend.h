// paged_attend.h -- attention over a paged key/value cache whose sequences may share their first positions:
// the kernel, built for one head_dim a translation unit.
#pragma once

#include "mla.h"
#include "paged.h"

namespace jero {

// What places that hold nothing are read from: 8 values of either type.
__device__ __constant__ const uint32_t kPagedZeros[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};

// The swap of a row's 16-byte chunks in LDS, chunk k of row r at k ^ swap(r): f16 rows of HD.  LDS has 64 banks of 4 bytes.  A
// read of 16 bytes a lane goes by 16 lanes: those of 8 rows at one chunk and of the 8 others at the next (lanes 0 - 3,
// 12 - 15 and 20 - 27, then 4 - 11, 16 - 19 and 28 - 31); a transposing read by 32, two chunks of 8 rows.  Neither meets on
// a bank: rows of 256 bytes and more have 16 chunks to swap, rows of 128 two to a round of the banks.  (Swaps within 128
// bytes: 2 ways, and chunks of nine prompts took 635 us.)  It is linear in the row's bits, so that a swap by a constant is
// one more exclusive or.
template <int HD>
__host__ __device__ __forceinline__ constexpr int swap_of(int r) {
  const int x = HD == 64 ? r >> 1 : r;
  return HD == 64 ? ((x & 3) << 1) ^ ((x & 4) ? 5 : 0) : ((x & 7) << 1) ^ ((x & 8) ? 9 : 0);
}

// ---------------------------------------------------------------- what a workgroup works on

// Starts that a workgroup copies to LDS for its searches: 7 steps there instead of 7 times the memory's latency (23
// sequences of 3 and 4 tokens behind 4608 positions: 29 us and 23).
constexpr int kSearchSeqs = 1024;
__device__ __forceinline__ const int32_t* paged_starts(const PagedCall& c, int32_t* s_starts, int tid) {
  if (!c.starts || c.n_seqs > kSearchSeqs) return c.starts;
  for (int i = tid; i <= c.n_seqs; i += 256) s_starts[i] = c.starts[i];
  __syncthreads();
  return s_starts;
}

// Position below which token row t of the call attends (t's own and max_len within it), by every lane on its own; -1: no
// sequence's.
__device__ __forceinline__ int paged_visible(const PagedCall& c, const int32_t* starts, int t) {
  int seq = t, end = t + 1;
  if (c.starts) {
    int lo = 0, left = c.n_seqs + 1;  // starts from 0 .. lo - 1 are not behind t
    while (left > 0) {
      const int half = left >> 1;
      if (starts[lo + half] <= t) lo += half + 1, left -= half + 1;
      else left = half;
    }
    seq = lo - 1;
    if (seq < 0 || seq >= c.n_seqs) return -1;
    end = starts[seq + 1];
  }
  const int64_t pos = int64_t(c.lens[seq]) - end + t;
  return int(max(min(pos + 1, int64_t(c.max_len)), int64_t(0)));
}

// Rows (token row * group + head of the group) first .. first + count - 1 of the kv head, the positions lo .. hi - 1,
// and the sequence whose table holds those that are not shared.
struct PagedItem {
  int first, count, lo, hi, seq, head, part;
  int end;        // own positions: the token row behind the sequence's last, by which hi is still to be bounded; or -1
  int64_t shift;  // and then the position of token row t is shift + t
};

__device__ __forceinline__ bool paged_item(const PagedCall& c, const PagedPlan& p, int lane, PagedItem& it, bool& wide) {
  // the two phases' blocks by turns, 256 of each: a CU gets one that computes and one that reads
  const int k = blockIdx.x >> 8, in = blockIdx.x & 255;
  const int np = (p.pre_blocks + 255) >> 8, no = (p.own_blocks + 255) >> 8, both = min(np, no);
  const bool pre = k < 2 * both ? (k & 1) == 0 : np > no;
  const int i = (k < 2 * both ? k >> 1 : k - both) * 256 + in;
  if (i >= (pre ? p.pre_blocks : p.own_blocks)) return false;
  it.head = i % c.kv_heads;
  const int rest = i / c.kv_heads;
  if (pre) {
    const int tile = rest % p.pre_tiles, chunk = rest / p.pre_tiles;
    const int rows = p.pre_wide ? p.wide_rows : kNarrowRows;
    wide = p.pre_wide;
    it.first = tile * rows;
    it.count = min(rows, c.n_tokens * c.group - it.first);
    it.lo = chunk * p.pre_len;
    it.hi = min(it.lo + p.pre_len, c.shared_len);
    it.seq = 0, it.part = chunk, it.end = -1;
    return true;
  }
  wide = p.own_wide;
  const int rows = wide ? p.wide_rows : kNarrowRows;
  const int chunk = rest / p.own_tiles, tile = p.own_tiles - 1 - rest % p.own_tiles;
  int end, from, skip = 0;
  if (!c.starts) {
    // a token's tiles
    const int each = (c.group + rows - 1) / rows;
    it.seq = tile / each, skip = tile % each * rows;
    from = it.seq, end = it.seq + 1;
  } else {
    // sequence s holds tiles floor(starts[s] group / rows) + s on: enough for its rows, and they do not fall with s
    int count = 0, left = c.n_seqs;  // sequences 0 .. count - 1 begin at no later tile
    while (left > 0) {
      const int step = (left + kWave - 1) / kWave, j = count + lane * step + step - 1;
      const int s = min(j, c.n_seqs - 1);
      const int64_t at = int64_t(min(max(c.starts[s], 0), c.n_tokens)) * c.group / rows + s;
      const int n = __popcll(__ballot(j < count + left && at <= tile));
      const int past = n * step;
      left = min(step - 1, left - past);
      count += past;
    }
    it.seq = count - 1;
    if (it.seq < 0) return false;
    from = min(max(c.starts[it.seq], 0), c.n_tokens);
    end = c.starts[it.seq + 1];
    skip = int(tile - (int64_t(from) * c.group / rows + it.seq)) * rows;
  }
  const int mine = max(min(end, c.n_tokens) - from, 0) * c.group;
  if (skip < 0 || skip >= mine) return false;
  it.first = from * c.group + skip;
  it.count = min(rows, mine - skip);
  it.lo = p.own_lo + chunk * p.own_len;
  it.hi = it.lo + p.own_len;
  it.end = end;
  it.part = p.pre_chunks + chunk;
  return true;
}

// Bounds hi by what the last row sees; false: no position is left, and no one else waits for the rows.
__device__ __forceinline__ bool paged_bound(const PagedCall& c, const PagedPlan& p, PagedItem& it) {
  if (it.end < 0) return true;
  const int last = (it.first + it.count - 1) / c.group;
  it.shift = int64_t(c.lens[it.seq]) - it.end;
  const int64_t top = min(it.shift + last + 1, int64_t(c.max_len));
  it.hi = int(max(min(top, int64_t(it.hi)), int64_t(it.lo)));
  return p.parts == 1 || it.hi > it.lo;  // (the only part of a row writes it whatever it sees)
}

// ---------------------------------------------------------------- a wave's step

template <int HD, int NJ, bool TWOQ>
struct AttendState {
  static constexpr int KT = HD / 32, DT = HD / 16;
  h8_t qh[NJ][KT], ql[NJ][TWOQ ? KT : 1];
  f4_t o[NJ][DT], l[NJ];
  float factor[NJ], m[NJ];
  int limit[NJ];  // positions below it are seen by the lane's row
};

constexpr float kPagedLift = 11.f, kPagedGrow = 4.f;

// KR positions from p0 on: S^T = K q^T leaves a row per lane column and, taken in the order 4g .. 4g + 3, 16 + 4g .. of
// 32 positions, is the B operand of O^T += V^T p, V^T read from LDS transposed.  ok: positions that are there; bad:
// those whose values are not finite and have been made zeros.  kread and vread give the products' operands; after_keys and
// before_values are done in between.  EARLY: the values are in LDS from the start.
template <int HD, int NJ, int KR, bool TWOQ, bool TWOK, bool EARLY, typename KRead, typename VRead, typename AfterKeys,
          typename BeforeValues>
__device__ __forceinline__ void attend_step(AttendState<HD, NJ, TWOQ>& st, KRead kread, VRead vread, AfterKeys after_keys,
                                            BeforeValues before_values, int p0, bool masked, uint64_t ok, uint64_t bad, int g) {
  constexpr int RT = KR / 16, KT = HD / 32, DT = HD / 16, KP = TWOK ? 2 : 1;
  f4_t s[NJ][RT];
  constexpr int KD = !EARLY ? 1 : RT == 2 ? 3 : 2;  // (registers; where values come late, keys are in them)
  h8_t ka[KD][RT][KP];
  auto read_k = [&](int k) {
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int e = 0; e < KP; e++) ka[k % KD][r][e] = kread(k, r, e);
  };
#pragma unroll
  for (int k = 0; k < KD - 1; k++) read_k(k);
#pragma unroll
  for (int k = 0; k < KT; k++) {
    if (KD == 1) read_k(k);
    else if (k + KD - 1 < KT) read_k(k + KD - 1);
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int j = 0; j < NJ; j++)
        s[j][r] = mfma(ka[k % KD][r][0], st.qh[j][k], k ? s[j][r] : f4_t{0.f, 0.f, 0.f, 0.f});
    if constexpr (TWOQ) {
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int j = 0; j < NJ; j++) s[j][r] = mfma(ka[k % KD][r][0], st.ql[j][k], s[j][r]);
    }
    if constexpr (TWOK) {
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int j = 0; j < NJ; j++) s[j][r] = mfma(ka[k % KD][r][KP - 1], st.qh[j][k], s[j][r]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  after_keys();
  // the values' first operands are on their way during the softmax
  constexpr int VD = 3;
  h8_t va[VD][RT / 2][KP];
  auto read_v = [&](int d) { vread(d, va[d % VD]); };
  if constexpr (EARLY)
#pragma unroll
    for (int d = 0; d < VD - 1; d++) read_v(d);
  h8_t bh[NJ][RT / 2], bl[NJ][RT / 2];
  bool grew[NJ];
  float alpha[NJ], times[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) times[j] = st.factor[j];
  if (masked) {
    const uint64_t mine = ok >> (4 * g), odd = bad >> (4 * g);
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      times[j] = 1.f;
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint64_t bit = 1ull << (16 * r + e);
          const float y = (odd & bit) ? NAN : s[j][r][e] * st.factor[j];
          s[j][r][e] = p0 + 16 * r + 4 * g + e < st.limit[j] && (mine & bit) ? y : -INFINITY;
        }
    }
  }
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    float mx = s[j][0][0];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[j][r][e]);
    mx = max_over_groups(mx) * times[j];
    grew[j] = __any(mx > st.m[j] + kPagedGrow);
    const float mn = grew[j] ? fmaxf(st.m[j], mx) : st.m[j];
    const float ref = mn == -INFINITY ? 0.f : mn, from = ref - kPagedLift;
    alpha[j] = __builtin_amdgcn_exp2f(st.m[j] - ref);
    st.m[j] = mn;
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[j][r][e], times[j], -from));
        _Float16 a, b;
        split2(p, a, b);
        bh[j][r / 2][4 * (r & 1) + e] = a;
        bl[j][r / 2][4 * (r & 1) + e] = b;
      }
  }
#pragma unroll
  for (int j = 0; j < NJ; j++)
    if (grew[j]) {
      st.l[j] *= alpha[j];
#pragma unroll
      for (int d = 0; d < DT; d++) st.o[j][d] *= alpha[j];
    }
  // the sums of the numerators, as the product rounds them: a row of ones in place of the values
  {
    h8_t one;
#pragma unroll
    for (int e = 0; e < 8; e++) one[e] = _Float16(1.f);
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int r = 0; r < RT / 2; r++) {
        st.l[j] = mfma(one, bh[j][r], st.l[j]);
        if constexpr (TWOQ) st.l[j] = mfma(one, bl[j][r], st.l[j]);
      }
  }
  if constexpr (!EARLY) {
    before_values();
#pragma unroll
    for (int d = 0; d < VD - 1; d++) read_v(d);
  }
#pragma unroll
  for (int d = 0; d < DT; d++) {
    if (d + VD - 1 < DT) read_v(d + VD - 1);
#pragma unroll
    for (int r = 0; r < RT / 2; r++) {
#pragma unroll
      for (int j = 0; j < NJ; j++) st.o[j][d] = mfma(va[d % VD][r][0], bh[j][r], st.o[j][d]);
      if constexpr (TWOQ) {
#pragma unroll
        for (int j = 0; j < NJ; j++) st.o[j][d] = mfma(va[d % VD][r][0], bl[j][r], st.o[j][d]);
      }
      if constexpr (TWOK) {
#pragma unroll
        for (int j = 0; j < NJ; j++) st.o[j][d] = mfma(va[d % VD][r][KP - 1], bh[j][r], st.o[j][d]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

typedef __attribute__((address_space(3))) h8_t lds_h8;

// Where a lane reads: keys' rows 16 r + col from chunk g on, values' rows 4 g + (col >> 2) transposed; then 64 bytes of the row
// further for each k, 32 for each d, within 256 by an exclusive or.
template <int HD>
__device__ __forceinline__ uint32_t key_lane(int g, int col) {
  return uint32_t(col * HD * 2 + 16 * (g ^ swap_of<HD>(col)));
}
template <int HD>
__device__ __forceinline__ uint32_t value_lane(int g, int col) {
  const int r = 4 * g + (col >> 2);
  return uint32_t(r * HD * 2 + 16 * (((col & 3) >> 1) ^ swap_of<HD>(r)) + 8 * (col & 1));
}
// Columns 16 d + col of the values of 32 N positions, as A operands: rows of f16 (in PARTS planes) read transposed.
template <int HD, int N, int PARTS>
__device__ __forceinline__ void read_transposed(uint32_t at, int plane, int d, h8_t (&to)[N][PARTS]) {
  const uint32_t p = (at ^ (32 * (d & 7))) + 256 * (d >> 3);
#pragma unroll
  for (int r = 0; r < N; r++)
#pragma unroll
    for (int e = 0; e < PARTS; e++) {
      const uint32_t q = p + e * plane + 32 * r * HD * 2;
      const s4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)uintptr_t(q));
      const s4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)uintptr_t(q + 16 * HD * 2));
      to[r][e] = __builtin_bit_cast(h8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// ---------------------------------------------------------------- the kernel

// out = sum_j softmax_j(scale q . k_j) v_j in one pass with a running maximum and sum, for two kinds of tiles.
//
// F ("wide"): many rows over the same positions.  Four waves share KR positions in LDS, up to three steps of them on their
// way, and hold 16 NJ rows each.  Bound by the products and the softmax between them: products busy 43 % and other vector
// instructions 40 % of the cycles.  Chunks of nine prompts, 6823 tokens behind 4096 shared positions, 32 heads of 128
// over 4, f16: 626 to 680 us over cards, 840 to 910 TFLOP/s of what the mask leaves; f32 activations, two products for one,
// 1080; over an f32 cache, three and the parts made in registers, 2260.  64 positions a step and two buffers: 32 and four
// 14 % more; the softmax of one half under the products of the other, with its maxima taken twice, 8 % more; wave priorities
// nothing.  Timed without the exponentials 5 % less, without loads 15 % less.
//
// D ("narrow"): a token's rows, or a few tokens'.  Four waves share 16 rows and hold 32 positions each, keys in registers,
// values in their own part of LDS, both asked for a step ahead; the waves are joined at the end.  Bound by the cache's bytes:
// 64 sequences of 6144 positions, 8 heads of 128, f16: 285 us, 5.65 TB/s; of 1536 79 us, 5.1 TB/s; one of 131072 110 us, 4.9.
// 32 rows a tile: registers spill, 16 sequences of 5 to 8 tokens and 4 heads 47 us against 36.
//
// Both are one launch, 256 workgroups of each by turns: where the shared positions make no more than 256, a CU gets one that
// computes and one that reads (64 f32 chats of 30 to 1500 positions behind 8192: shared positions alone 45 us, own alone 47,
// the call 61).  More of them fill both places of a CU, and most own positions come after (256 f16 chats of 10 to 700
// behind 32768, 512 workgroups: 297 and 100, the call 362).
//
// f16 activations: numerators are one f16 part, where everything else is as exact as the f16 inputs.  Results are off by 2.5e-4
// to 2.8e-4 of their size, of which their own rounding is 2.1e-4.  A second part for them leaves that rounding alone and takes
// 30 to 36 % more: those 256 chats 455 us for 350, the chunks of nine prompts 851 for 628.
template <int HD, typename X, typename KV>
struct PagedShape {
  static constexpr bool TWOQ = sizeof(X) == 4, TWOK = sizeof(KV) == 4;
  static constexpr int NJ = HD <= 128 && !TWOK ? 2 : 1, KR = TWOQ || HD == 256 ? 32 : 64;
  static constexpr int kRows = 64 * NJ;
  static constexpr int kPlanes = TWOK ? 2 : 1;
  static constexpr int kPlane = KR * HD * 2, kBuf = 2 * kPlanes * kPlane;  // keys, then values
  static constexpr int kBufs = TWOK ? 1 : HD == 256 ? 4 : 64 * 1024 / kBuf > 4 ? 4 : 64 * 1024 / kBuf;
  static constexpr int kNarrow = 32 * HD * int(sizeof(KV));                // a wave's values
  static constexpr int kValueBufs = TWOK && HD > 64 ? 1 : 2;
  static constexpr int kWaveLds = kNarrow * kValueBufs;
  static constexpr int kJoin = 4 * 16 * (HD + 4) * 4;
  static constexpr int kMost = kBufs * kBuf > 4 * kWaveLds ? kBufs * kBuf : 4 * kWaveLds;
  static constexpr int kLds = kMost > kJoin ? kMost : kJoin;
  static constexpr int kGroups = HD == 256 ? 1 : 2;
};

// Whether 16 bytes of values have one that is not finite as f16: the exponent's bits all set, or an f32 that rounds past 65504.
template <typename KV>
__device__ __forceinline__ bool odd_piece(u32x4 v) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t w = v[i];
    if constexpr (sizeof(KV) == 4) odd |= !(fabsf(__uint_as_float(w)) < 65520.f);
    else odd |= (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
  }
  return odd;
}

template <int HD, typename X, typename KV>
__global__ void __launch_bounds__(256, (PagedShape<HD, X, KV>::kGroups))
    paged_attend_kernel(PagedCall c, PagedPlan plan, const X* __restrict__ q, X* __restrict__ out,
                        float* __restrict__ part_o, float2* __restrict__ part_ml) {
  using S = PagedShape<HD, X, KV>;
  constexpr bool TWOQ = S::TWOQ, TWOK = S::TWOK;
  constexpr int KT = HD / 32, DT = HD / 16;
  __shared__ __attribute__((aligned(256))) uint8_t s_kv[S::kLds];
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_low;
  __shared__ int32_t s_starts[kSearchSeqs + 1];
  __shared__ unsigned long long s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  PagedItem it;
  bool wide;
  if (!paged_item(c, plan, lane, it, wide)) return;
  const uint32_t lds0 = uint32_t(uintptr_t((lds_u8*)s_kv));
  const int D = c.dim;
  const int64_t row_len = int64_t(c.kv_heads) * D;
  const KV* const kb = static_cast<const KV*>(c.k) + int64_t(it.head) * D;
  const KV* const vb = static_cast<const KV*>(c.v) + int64_t(it.head) * D;
  const int32_t* const table = c.table + it.seq * c.table_stride;
  const void* const zeros = kPagedZeros;
  // A load to LDS of 1024 bytes holds RPI rows.  Where all positions of a step are there and blocks hold that many, its
  // rows follow each other from one address for the whole wave (values behind head_dim are then the row's first: no
  // query's, and not stored).
  constexpr int RPI = 1024 / (2 * HD);
  const int shift_mask = (1 << c.shift) - 1;
  const int64_t row_bytes = row_len * int64_t(sizeof(KV)), block_bytes = row_bytes << c.shift;
  auto offset_of = [&](uint32_t ids, int r, int p0) -> int64_t {  // of row r of a step, the wave's
    const uint32_t id = __builtin_amdgcn_readlane(ids, r);
    return int64_t(id) * block_bytes + int64_t((p0 + r) & shift_mask) * row_bytes;
  };

  // The block of the lane's position of a step from p0 on; ~0: none, or not the item's.  64 blocks' ids are kept, a lane
  // each, and the load that renews them is waited for where it is made: a wait further on would be for all loads in flight.
  uint32_t window = ~0u;
  int window0 = INT32_MIN / 2;
  auto open_window = [&](int b0) {
    window0 = b0;
    const int b = b0 + lane;
    window = ~0u;
    if (b < c.table_stride) window = uint32_t(b < c.shared_blocks ? c.shared[b] : table[b]);
  };
  auto blocks_of = [&](int p0, int kr) -> uint32_t {
    const int b0 = p0 >> c.shift;
    if (b0 - window0 >= kWave) {
      open_window(b0);
      asm volatile("" : "+v"(window));
      window = window < c.n_blocks ? window : ~0u;
    }
    const int pos = p0 + (lane & (kr - 1));
    const uint32_t id = __shfl(window, (pos >> c.shift) - window0, kWave);
    return pos < it.hi ? id : ~0u;
  };
  auto row_of = [&](const KV* base, uint32_t id, int pos) -> const uint8_t* {
    return reinterpret_cast<const uint8_t*>(base + ((int64_t(id) << c.shift) + (pos & ((1 << c.shift) - 1))) * row_len);
  };
  const uint32_t value0 = value_lane<HD>(g, col);

  // Positions that a token of the item sees: those of its sequence, or found for each.
  const int32_t* const starts = it.end < 0 ? paged_starts(c, s_starts, tid) : nullptr;
  auto visible = [&](int t) {
    if (it.end < 0) return paged_visible(c, starts, t);
    return int(max(min(it.shift + t + 1, int64_t(c.max_len)), int64_t(0)));
  };
  // The queries of the lane's columns, from the wave's row `row0` on: their loads, which hang on no length (rows of no
  // sequence are not read), then what is made of them.
  int owned_lo = 0, owned_hi = c.n_tokens;
  if (c.starts && it.end < 0) owned_lo = c.starts[0], owned_hi = c.starts[c.n_seqs];
  constexpr int QW = TWOQ ? 2 : 1;
  auto load_queries = [&](auto& raw, int row0) {
    constexpr int NJ = sizeof(raw) / (KT * QW * 16);
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int i = row0 + 16 * j + col, r = it.first + (i < it.count ? i : 0), t = r / c.group;
      const X* qr = q + t * c.q_stride + int64_t(it.head * c.group + r % c.group) * D;
#pragma unroll
      for (int k = 0; k < KT; k++) {
        const int d = 32 * k + 8 * g;
        const bool on = d < D && t >= owned_lo && t < owned_hi;
        const uint8_t* p = on ? reinterpret_cast<const uint8_t*>(qr + d) : static_cast<const uint8_t*>(zeros);
#pragma unroll
        for (int e = 0; e < QW; e++) raw[j][k][e] = *reinterpret_cast<const u32x4*>(p + 16 * e);
      }
    }
  };
  auto queries = [&](auto& st, const auto& raw, int row0) {
    constexpr int NJ = sizeof(st.m) / sizeof(float);
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int i = row0 + 16 * j + col;
      const bool mine = i < it.count;
      const int seen = mine ? visible((it.first + i) / c.group) : 0;
      st.limit[j] = seen;
      float v[KT][8], mx = 0.f;
#pragma unroll
      for (int k = 0; k < KT; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          float x;
          if constexpr (TWOQ) x = __uint_as_float(raw[j][k][e >> 2][e & 3]);
          else x = float(__builtin_bit_cast(h8_t, raw[j][k][0])[e]);
          v[k][e] = seen > 0 ? x : 0.f;
          mx = fmaxf(mx, fabsf(v[k][e]));
        }
      // each row's brought near 1 by a power of two that goes into the scores' factor
      mx = max_over_groups(mx);
      int ex = 0;
      if (TWOQ && mx > 0.f && mx < INFINITY) ex = ilogbf(mx);
      st.factor[j] = ldexpf(fabsf(c.scale) * 1.44269504088896341f, ex);  // its sign goes into the queries
#pragma unroll
      for (int k = 0; k < KT; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          _Float16 a, b;
          split2(ldexpf(c.scale < 0.f ? -v[k][e] : v[k][e], -ex), a, b);
          st.qh[j][k][e] = a;
          if (TWOQ) st.ql[j][k][e] = b;
        }
      st.m[j] = -INFINITY;
      st.l[j] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DT; d++) st.o[j][d] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
  };
  // Lowest limit of the wave's rows that see anything (those that do not are put right at the end).
  auto lowest = [&](const auto& st) {
    constexpr int NJ = sizeof(st.m) / sizeof(float);
    int low = INT32_MAX;
#pragma unroll
    for (int j = 0; j < NJ; j++) low = min(low, st.limit[j] > 0 ? st.limit[j] : INT32_MAX);
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) low = min(low, __shfl_xor(low, off, kWave));
    return low;
  };
  // Row i of the item, 4 of its results.
  auto store = [&](int i, int d, f4_t v, float m, float l, bool first) {
    const int r = it.first + i, t = r / c.group, h = it.head * c.group + r % c.group;
    if (plan.parts > 1) {
      const int64_t at = (int64_t(it.part) * c.n_tokens + t) * c.heads + h;
      if (d < D) *reinterpret_cast<f4_t*>(part_o + at * D + d) = v;
      if (first) part_ml[at] = make_float2(m, l);
      return;
    }
    if (d >= D) return;
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    X* dst = out + t * c.out_stride + int64_t(h) * D + d;
    if constexpr (sizeof(X) == 4) {
      *reinterpret_cast<f4_t*>(dst) = v * inv;
    } else {
      h4_t y;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = _Float16(v[e] * inv);
      *reinterpret_cast<h4_t*>(dst) = y;
    }
  };

  if (wide) {
    // ------------------------------------------------------------ F
    constexpr int KR = S::KR, NJ = S::NJ;
    AttendState<HD, NJ, TWOQ> st;
    if (tid == 0) s_low = INT32_MAX, s_bad = 0;
    open_window(it.lo >> c.shift);
    u32x4 qraw[NJ][KT][QW];
    load_queries(qraw, wv * 16 * NJ);
    if (!paged_bound(c, plan, it)) return;
    window = window < c.n_blocks ? window : ~0u;
    queries(st, qraw, wv * 16 * NJ);
    const int low = lowest(st);
    __syncthreads();
    if (lane == 0) atomicMin(&s_low, low);
    __syncthreads();
    const int common = s_low;  // below it, all rows of the workgroup see a position
    const int steps = (it.hi - it.lo + KR - 1) / KR;
    constexpr int NI = S::kPlane / 1024 / 4;  // 1024-byte pieces a wave, of keys and of values
    const int lane_row = lane / (HD / 8);
    const int lane_at = (16 * lane) % (2 * HD) ^ (16 * swap_of<HD>(wv * RPI + lane_row));
    auto piece_at = [&](int n) { return lane_at ^ (16 * swap_of<HD>(4 * n * RPI)); };  // piece 4 n + wv
    auto load = [&](int step, int buf, uint32_t ids) {  // f16: straight to LDS
      const int p0 = it.lo + step * KR;
      if (__ballot(ids != ~0u) == ~0ull && (1 << c.shift) >= RPI) {
#pragma unroll
        for (int n = 0; n < NI; n++) {
          const int i = 4 * n + wv;
          const int64_t at = offset_of(ids, i * RPI, p0);
          const uint32_t to = lds0 + buf * S::kBuf + i * 1024;
          const uint32_t lane_bytes = uint32_t(lane_row * row_bytes) + (piece_at(n) < 2 * D ? piece_at(n) : 0);
          dma_row(reinterpret_cast<const uint8_t*>(kb) + at, lane_bytes, to);
          dma_row(reinterpret_cast<const uint8_t*>(vb) + at, lane_bytes, to + S::kPlane);
        }
        return;
      }
#pragma unroll
      for (int n = 0; n < NI; n++) {
        const int i = 4 * n + wv, r = i * RPI + lane_row, at = piece_at(n);
        const uint32_t id = __shfl(ids, r, kWave);
        const bool on = id != ~0u && at < 2 * D;
        const uint32_t to = lds0 + buf * S::kBuf + i * 1024;
        dma_lanes(on ? row_of(kb, id, p0 + r) + at : zeros, to);
        dma_lanes(on ? row_of(vb, id, p0 + r) + at : zeros, to + S::kPlane);
      }
    };
    // f32: through registers, a lane 8 values of a row
    constexpr int NR = TWOK ? KR * HD / 8 / 256 : 1;
    float raw[TWOK ? 2 : 1][NR][8];
    auto fetch = [&](int step, uint32_t ids) {
      const int p0 = it.lo + step * KR;
#pragma unroll
      for (int n = 0; n < NR; n++) {
        const int i = n * 256 + tid, r = i / (HD / 8), d = 8 * (i % (HD / 8));
        const uint32_t id = __shfl(ids, r, kWave);
        const bool on = id != ~0u && d < D;
        load8<float>(static_cast<const float*>(on ? static_cast<const void*>(row_of(kb, id, p0 + r) + 4 * d) : zeros), raw[0][n]);
        load8<float>(static_cast<const float*>(on ? static_cast<const void*>(row_of(vb, id, p0 + r) + 4 * d) : zeros),
                     raw[TWOK ? 1 : 0][n]);
      }
    };
    auto put = [&]() {
#pragma unroll
      for (int w = 0; w < (TWOK ? 2 : 1); w++)
#pragma unroll
        for (int n = 0; n < NR; n++) {
          const int i = n * 256 + tid, r = i / (HD / 8), d = i % (HD / 8);
          h8_t hi, lo;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            _Float16 a, b;
            split2(raw[w][n][e], a, b);
            hi[e] = a, lo[e] = b;
          }
          uint8_t* to = s_kv + w * S::kPlanes * S::kPlane + r * HD * 2 + 16 * (d ^ swap_of<HD>(r));
          *reinterpret_cast<h8_t*>(to) = hi;
          *reinterpret_cast<h8_t*>(to + S::kPlane) = lo;
        }
    };
    const uint32_t key0 = key_lane<HD>(g, col);
    // tiles on their way: A of them, each kLoads loads a wave; and which of their positions are there
    constexpr int A = TWOK ? 1 : S::kBufs - 1, kLoads = 2 * NI;
    uint64_t there[A];
    auto ask = [&](int i, int to) -> uint64_t {
      if (i >= steps) return 0;
      const uint32_t ids = blocks_of(it.lo + i * KR, KR);
      if constexpr (TWOK) fetch(i, ids);
      else load(i, to, ids);
      return __ballot(ids != ~0u);
    };
#pragma unroll
    for (int i = 0; i < A; i++) there[i] = ask(i, i);
    int buf = 0;
    for (int i = 0; i < steps; i++) {
      const int p0 = it.lo + i * KR;
      const uint64_t ok = there[0];
#pragma unroll
      for (int n = 0; n + 1 < A; n++) there[n] = there[n + 1];
      if constexpr (TWOK) {
        __syncthreads();  // the last step's reads
        put();
        __syncthreads();
        there[0] = ask(i + 1, 0);
      } else {
        if (i + A <= steps) dma_wait<(A - 1) * kLoads>();
        else dma_wait<0>();
        __syncthreads();  // (and the last step's reads are done: its buffer is the next to be filled)
        there[A - 1] = ask(i + A, buf == 0 ? A : buf - 1);
      }
      uint8_t* const kv = s_kv + buf * S::kBuf;
      uint64_t bad = 0;
      if (min(p0 + KR, it.hi) > common) {
        // Values that are not finite, of which a row that does not see them would take 0 * infinity, are made zeros, and
        // their positions' scores NaN.
        constexpr int L = HD / 8;
        uint8_t* const rows = kv + S::kPlanes * S::kPlane;
        for (int n = tid; n < KR * L; n += 256)
          if (odd_piece<_Float16>(*reinterpret_cast<const u32x4*>(rows + 16 * n))) atomicOr(&s_bad, 1ull << (n / L));
        __syncthreads();
        bad = s_bad;
        if (bad) {
          const u32x4 z = {0u, 0u, 0u, 0u};
          for (int n = tid; n < KR * L; n += 256)
            if ((bad >> (n / L)) & 1) {
              *reinterpret_cast<u32x4*>(rows + 16 * n) = z;
              if (TWOK) *reinterpret_cast<u32x4*>(rows + S::kPlane + 16 * n) = z;
            }
        }
        __syncthreads();
        if (tid == 0) s_bad = 0;  // (the next step's barriers come before its next use)
      }
      const uint32_t at = lds0 + buf * S::kBuf;
      auto kread = [&](int k, int r, int e) {
        const uint32_t p = ((at + key0) ^ (64 * (k & 3))) + 256 * (k >> 2);
        return *(lds_h8*)uintptr_t(p + e * S::kPlane + 16 * r * HD * 2);
      };
      auto vread = [&](int d, auto& to) {
        read_transposed<HD, KR / 32, S::kPlanes>(at + S::kPlanes * S::kPlane + value0, S::kPlane, d, to);
      };
      // (bad: a wave whose rows all see the step has been given zeros for its values too)
      const bool masked = bad || p0 + KR > low || ok != ~0ull || p0 + KR > it.hi;
      auto none = [] {};
      attend_step<HD, NJ, KR, TWOQ, TWOK, true>(st, kread, vread, none, none, p0, masked, ok, bad, g);
      if (!TWOK) buf = buf == S::kBufs - 1 ? 0 : buf + 1;
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int i = wv * 16 * NJ + 16 * j + col;
      if (i >= it.count || st.limit[j] < 0) continue;
      const bool sees = st.limit[j] > it.lo;
      const f4_t z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DT; d++)
        store(i, 16 * d + 4 * g, sees ? st.o[j][d] : z, sees ? st.m[j] : -INFINITY, sees ? st.l[j][0] : 0.f, d == 0 && g == 0);
    }
    return;
  }

  // -------------------------------------------------------------- D
  constexpr int KR = 32;
  AttendState<HD, 1, TWOQ> st;
  open_window(it.lo >> c.shift);
  u32x4 qraw[1][KT][QW];
  load_queries(qraw, 0);
  if (!paged_bound(c, plan, it)) return;
  window = window < c.n_blocks ? window : ~0u;
  const int steps = (it.hi - it.lo + KR - 1) / KR;
  uint8_t* const mine = s_kv + wv * S::kWaveLds;
  const uint32_t mine0 = lds0 + wv * S::kWaveLds;
  constexpr int KRAW = TWOK ? 2 : 1;  // 16-byte pieces for 8 values
  u32x4 kraw[2][KT][KRAW];            // keys: row 16 r + col, values 32 k + 8 g ..
  // Values go straight to LDS, pieces of 1024 bytes.  f32 rows are swapped by 64 bytes, by (r >> 2) & 3: the four rows that a
  // read wants at once, 4 apart, are then on banks of their own.
  constexpr int VR = 1024 / (HD * int(sizeof(KV))), PIECES = 32 / VR;
  const int lane_row = lane / (64 / VR);
  const int lane_at = 16 * lane % (1024 / VR) ^ (TWOK ? 0 : 16 * swap_of<HD>(lane_row));
  auto value_at = [&](int i) {  // byte of the row that the lane loads of piece i
    return lane_at ^ (TWOK ? 64 * ((i * VR >> 2) & 3) : 16 * swap_of<HD>(i * VR));
  };
  constexpr int kKeyLoads = 2 * KT * KRAW;
  auto fetch_values = [&](int step, int buf, uint32_t ids) {
    const int p0 = it.lo + step * KR, bytes = D * int(sizeof(KV));
    const uint32_t to = mine0 + buf * S::kNarrow;
    if (__ballot(ids != ~0u) == ~0ull && (1 << c.shift) >= VR) {
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int at = value_at(i);
        dma_row(reinterpret_cast<const uint8_t*>(vb) + offset_of(ids, i * VR, p0),
                uint32_t(lane_row * row_bytes) + (at < bytes ? at : 0), to + i * 1024);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      const int r = i * VR + lane_row, at = value_at(i);
      const uint32_t id = __shfl(ids, r, kWave);
      dma_lanes(id != ~0u && at < bytes ? row_of(vb, id, p0 + r) + at : zeros, to + i * 1024);
    }
  };
  auto fetch_keys = [&](int step, uint32_t ids) {
    const int p0 = it.lo + step * KR;
    if (__ballot(ids != ~0u) == ~0ull && c.shift >= 4) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const uint8_t* row = reinterpret_cast<const uint8_t*>(kb) + offset_of(ids, 16 * r, p0);
#pragma unroll
        for (int k = 0; k < KT; k++) {
          const int d = 32 * k + 8 * g;
          const uint32_t at = uint32_t(col * row_bytes) + (d < D ? d : 0) * int(sizeof(KV));
#pragma unroll
          for (int e = 0; e < KRAW; e++) kraw[r][k][e] = *reinterpret_cast<const u32x4*>(row + at + 16 * e);
        }
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const uint32_t id = __shfl(ids, 16 * r + col, kWave);
      const uint8_t* row = id != ~0u ? row_of(kb, id, p0 + 16 * r + col) : nullptr;
#pragma unroll
      for (int k = 0; k < KT; k++) {
        const int d = 32 * k + 8 * g;
        const bool on = row && d < D;
        const uint8_t* p = on ? row + d * int(sizeof(KV)) : static_cast<const uint8_t*>(zeros);
#pragma unroll
        for (int e = 0; e < KRAW; e++) kraw[r][k][e] = *reinterpret_cast<const u32x4*>(p + (on ? 16 * e : 0));
      }
    }
  };
  uint32_t ids = ~0u;
  if (wv < steps) {
    ids = blocks_of(it.lo + wv * KR, KR);
    fetch_values(wv, 0, ids);
    fetch_keys(wv, ids);
  }
  queries(st, qraw, 0);
  const int low = lowest(st);
  // Where LDS and registers hold two steps' values and keys, the next step's are asked for at a step's start; otherwise
  // when its own are used up.
  constexpr bool TWO_V = S::kValueBufs == 2, TWO_K = HD == 64 || !TWOK;
  int buf = 0;
  for (int i = wv; i < steps; i += 4) {
    const int p0 = it.lo + i * KR;
    const uint64_t ok = __ballot(ids != ~0u);
    const bool more = i + 4 < steps;
    uint8_t* const vp = mine + (TWO_V ? buf * S::kNarrow : 0);
    if (more) ids = blocks_of(p0 + 4 * KR, KR);
    if constexpr (TWO_V) {
      dma_wait<0>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last step's reads of the buffer that is loaded next
    }
    u32x4 kc[2][KT][KRAW];
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int k = 0; k < KT; k++)
#pragma unroll
        for (int e = 0; e < KRAW; e++) kc[r][k][e] = kraw[r][k][e];
    if (TWO_K && more) fetch_keys(i + 4, ids);
    if (TWO_V && more) fetch_values(i + 4, buf ^ 1, ids);
    const bool check = min(p0 + KR, it.hi) > low;
    if (!TWO_V && check) dma_wait<0>();
    uint64_t bad = 0;
    if (check) {
      constexpr int L = HD * int(sizeof(KV)) / 16;  // pieces of 16 bytes a row
      for (int n = lane; n < KR * L; n += 64) {
        const uint64_t b = __ballot(odd_piece<KV>(*reinterpret_cast<const u32x4*>(vp + 16 * n)));
#pragma unroll
        for (int x = 0; x < 64; x += L)
          if ((b >> x) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) bad |= 1ull << ((n - lane + x) / L);
      }
      if (bad) {
        const u32x4 z = {0u, 0u, 0u, 0u};
        for (int n = lane; n < KR * L; n += 64)
          if ((bad >> (n / L)) & 1) *reinterpret_cast<u32x4*>(vp + 16 * n) = z;
      }
    }
    const bool masked = p0 + KR > low || ok != ~0ull || p0 + KR > it.hi;
    auto kread = [&](int k, int r, int e) {
      if constexpr (!TWOK) {
        return __builtin_bit_cast(h8_t, kc[r][k][0]);
      } else {
        h8_t part;
#pragma unroll
        for (int x = 0; x < 8; x++) {
          _Float16 a, b;
          split2(__uint_as_float(kc[r][k][(KRAW - 1) * (x >> 2)][x & 3]), a, b);
          part[x] = e ? b : a;
        }
        return part;
      }
    };
    auto after_keys = [&] {
      if (!TWO_K && more) fetch_keys(i + 4, ids);
    };
    auto before_values = [&] {  // (the next keys' loads, behind the values', stay on their way)
      if (more) dma_wait<kKeyLoads>();
      else dma_wait<0>();
    };
    auto vread = [&](int d, auto& to) {
      if constexpr (!TWOK) {
        read_transposed<HD, 1, 1>(mine0 + uint32_t(vp - mine) + value0, 0, d, to);
      } else {
        const uint8_t* p = vp + 4 * g * HD * 4 + ((64 * g) ^ (64 * (d & 3))) + 256 * (d >> 2) + 4 * col;
        h8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          _Float16 x, y;
          split2(*reinterpret_cast<const float*>(p + ((e & 3) + 16 * (e >> 2)) * HD * 4), x, y);
          hi[e] = x, lo[e] = y;
        }
        to[0][0] = hi, to[0][TWOK ? 1 : 0] = lo;
      }
    };
    attend_step<HD, 1, KR, TWOQ, TWOK, TWO_V>(st, kread, vread, after_keys, before_values, p0, masked, ok, bad, g);
    if (!TWO_V && more) {  // (the one buffer is free when its reads are done)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      fetch_values(i + 4, 0, ids);
    }
    buf ^= 1;
  }
  // the four waves' rows joined
  float* const rows = reinterpret_cast<float*>(s_kv);
  if (g == 0) s_m[wv][col] = st.m[0], s_l[wv][col] = st.l[0][0];
  __syncthreads();
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; w++) m = fmaxf(m, s_m[w][col]);
  const float ref = m == -INFINITY ? 0.f : m, f = __builtin_amdgcn_exp2f(st.m[0] - ref);
#pragma unroll
  for (int d = 0; d < DT; d++)
    *reinterpret_cast<f4_t*>(rows + (wv * 16 + col) * (HD + 4) + 16 * d + 4 * g) = st.o[0][d] * f;
  __syncthreads();
  for (int n = tid; n < 16 * HD / 4; n += 256) {
    const int r = n / (HD / 4), d = 4 * (n % (HD / 4));
    if (r >= it.count) continue;
    const int seen = visible((it.first + r) / c.group);
    if (seen < 0) continue;
    const bool sees = seen > it.lo;
    float mm = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) mm = fmaxf(mm, s_m[w][r]);
    const float at = mm == -INFINITY ? 0.f : mm;
    f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; w++) {
      l += s_l[w][r] * __builtin_amdgcn_exp2f(s_m[w][r] - at);
      v += *reinterpret_cast<const f4_t*>(rows + (w * 16 + r) * (HD + 4) + d);
    }
    const f4_t z = {0.f, 0.f, 0.f, 0.f};
    store(r, d, sees ? v : z, sees ? mm : -INFINITY, sees ? l : 0.f, d == 0);
  }
}

template <int HD, typename X, typename KV>
static int launch_paged(const PagedCall& c, const PagedPlan& p, const void* q, void* out, float* part_o, float2* part_ml,
                        hipStream_t s) {
  const unsigned blocks = unsigned(((p.pre_blocks + 255) / 256 + (p.own_blocks + 255) / 256) * 256);
  hipLaunchKernelGGL((paged_attend_kernel<HD, X, KV>), dim3(blocks), dim3(256), 0, s, c, p, static_cast<const X*>(q),
                     static_cast<X*>(out), part_o, part_ml);
  return check_launch("paged_attention");
}

template <int HD>
static int launch_paged_types(const PagedCall& c, const PagedPlan& p, bool x16, bool kv16, const void* q, void* out,
                              float* part_o, float2* part_ml, hipStream_t s) {
  if (x16) return launch_paged<HD, _Float16, _Float16>(c, p, q, out, part_o, part_ml, s);
  if (kv16) return launch_paged<HD, float, _Float16>(c, p, q, out, part_o, part_ml, s);
  return launch_paged<HD, float, float>(c, p, q, out, part_o, part_ml, s);
}

}  // namespace jero
