// mla_prefill.hip -- latent attention over a paged cache: the expanded form, for prompts.
//
// For as many heads at a time as the workspace holds: mla_expand_kernel makes every position's keys and
// values, k = W_uk c and v = W_uv c, as rows of f16 (two parts a value with f32 activations), and copies
// the shared key parts next to each other; mla_flash_kernel runs the causal attention of 128 tokens of a
// sequence and a head over them.
#include "mla.h"

#include <type_traits>

namespace jero {

// Rows of the expanded keys and values: sequence s holds rows base(s) .. base(s) + min(lens[s],
// max_len) - 1, base the sum of the lengths before it that fit; one that would end past total has none.
__device__ __forceinline__ int mla_len(const LatentCache& c, int s) { return min(max(c.lens[s], 0), c.max_len); }

// Goes over the sequences, all lanes together: f(s, base, length) until it returns false.  Every workgroup does, so a
// call takes no more than kPrefillSeqs of them (2^19 tokens are then 2^13 tiles at most, 2^23 of 1024 heads).
constexpr int kPrefillSeqs = 4096;
template <typename F>
__device__ __forceinline__ void mla_sequences(const LatentCache& c, int64_t total, int lane, F f) {
  int64_t base = 0;
  for (int s0 = 0; s0 < c.n_seqs; s0 += kWave) {
    const int mine = s0 + lane < c.n_seqs ? mla_len(c, s0 + lane) : 0;
    const int n = min(kWave, c.n_seqs - s0);
    for (int j = 0; j < n; j++) {
      const int len = __builtin_amdgcn_readlane(mine, j);
      const bool fits = base + len <= total;
      if (!f(s0 + j, base, fits ? len : 0)) return;
      if (fits) base += len;
    }
  }
}

// The expanded rows: NT, PT, VT the padded widths; each part a plane of f16.
struct Expanded {
  _Float16 *k, *v, *p;  // [heads][total][NT], [heads][total][VT], [total][PT]
  uint8_t* odd;                       // [heads][total][VT / 64]: 64 values with one past f16's range
  int64_t k_plane, v_plane, p_plane;  // to the lower parts
  int64_t total;
};

// The product W C^T for 128 positions (64 of an f32 cache, whose latents go in as two f16 parts) and a run of the
// heads' padded weight rows (keys before values).  The latents stay in LDS for the whole run; a wave takes 64 weight
// rows at a time, their operands straight from memory (no other wave of the block wants them), so that each 1024
// bytes read from LDS serve four products.  A lane's rows of the four are chosen so that it ends up with 16
// consecutive columns of a position's row.  TWO: the results come out as two parts.  The last blocks copy the
// key parts.
//
// Measured: 4097 positions of 512 for 128 heads of 128 + 128 (f16): 214 us, 640 TFLOP/s and 270 MB written; 2048 for
// 32 heads, two parts: 41 us.  Bound by the products' issue and, with two parts, the rows written.  Steps before it:
// tiles of both operands in LDS 300 us, latents kept 225, weights' lines read whole 204.
template <typename KV>
struct ExpandShape {
  static constexpr bool kWide = sizeof(KV) == 4;
  static constexpr int kPos = kWide ? 64 : 128, kShort = 32, kPlanes = kWide ? 2 : 1;
  static constexpr int kPitch = kMlaMaxRank + 8;  // 16 rows fall on all banks
};
template <int NT, int PT, int VT, typename KV, bool TWO, int MP, int NW>
__global__ void __launch_bounds__(64 * NW) mla_expand_kernel(LatentCache c, int nh, int nope, int v_dim,
                                                         const _Float16* __restrict__ w, Expanded x, int run) {
  using S = ExpandShape<KV>;
  constexpr bool WIDE = S::kWide;
  constexpr int WP = NT + VT, CP = S::kPlanes, P = S::kPitch, MJ = MP / 16, JB = MJ < 4 ? MJ : 4;
  constexpr int STEP = 64 * NW;  // threads, and weight rows of the waves
  __shared__ __attribute__((aligned(16))) _Float16 s_c[CP][MP][P];
  // the positions' cache rows: -1 for a block that is none, -2 for no position; -3, once it is read, for one of
  // infinities or NaN
  __shared__ int64_t s_row[MP];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  // blocks of one run of weight rows follow each other, over all XCDs; the key parts' come last
  const int across = int((x.total + MP - 1) / MP), part = blockIdx.x / across;
  const int64_t m0 = int64_t(blockIdx.x % across) * MP;
  if (tid < (MP > kWave ? MP : kWave)) {  // (whole waves)
    int seq = -1, pos = 0;
    mla_sequences(c, x.total, lane, [&](int s, int64_t base, int len) {
      if (m0 + tid >= base && m0 + tid < base + len) seq = s, pos = int(m0 + tid - base);
      return base + len < m0 + MP;
    });
    if (tid < MP) s_row[tid] = seq < 0 ? -2 : mla_row(c, seq, pos);
  }
  __syncthreads();
  if (s_row[0] == -2) return;  // behind the last sequence's rows
  const KV* rows = static_cast<const KV*>(c.rows);

  if ((part + 1) * across == int(gridDim.x)) {
    for (int i = tid; i < MP * (PT / 8); i += STEP) {
      const int r = i / (PT / 8), k = 8 * (i % (PT / 8));
      const int64_t at = s_row[r];
      if (at == -2) continue;
      float v[8];
      if (at >= 0 && k < c.rope) load8<KV>(rows + at + c.rank + k, v);
      else
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
      h8_t hi, lo;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        _Float16 a, b;
        split2(v[e], a, b);
        hi[e] = a, lo[e] = b;
      }
      *reinterpret_cast<h8_t*>(x.p + (m0 + r) * PT + k) = hi;
      if (TWO) *reinterpret_cast<h8_t*>(x.p + x.p_plane + (m0 + r) * PT + k) = lo;
    }
    return;
  }

  const int g = lane >> 4, col = lane & 15;
  // weight row of the lane's operand of product i: the result's row 4g + e is column 16g + 4i + e
  const int all = nh * WP, w_end = min(all, (part + 1) * run);
  const _Float16* wp[4];
  auto rows_of = [&](int w0) {  // 64 of them belong to one head and one of its two parts
    const int h = w0 / WP, j = w0 % WP;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int n = (j < NT ? j : j - NT) + 16 * (col >> 2) + 4 * i + (col & 3);
      const bool on = w0 < w_end && (j < NT ? n < nope : n < v_dim);
      wp[i] = on ? w + (int64_t(h) * (nope + v_dim) + (j < NT ? n : nope + n)) * c.rank : nullptr;
    }
  };
  // Operands of 64 of the rank, two steps: a lane's 16 bytes of both follow each other in its row, so that both
  // loads want the same lines, whole, at once (taken in the row's order a wave's halves of lines come back to the
  // cache after eight waves have been through it)
  h8_t a[2][4][2];
  const int pairs = (c.rank + 63) / 64;
  auto read_w = [&](int p, h8_t (&d)[4][2]) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const int at = min(64 * p + 16 * g + 8 * s, c.rank - 8);  // (past the rank the latents are zeros)
        const h8_t z = {};
        d[i][s] = wp[i] ? *reinterpret_cast<const h8_t*>(wp[i] + at) : z;
      }
  };
  int w0 = part * run + 64 * wv;
  rows_of(w0);
  read_w(0, a[0]);

  // The latents: a lane 8 values, up to 8 rows' loads at a time.  A row that is not finite gets keys of NaN, which make
  // NaN of every token that attends to it, and values of zeros, as tokens before it would take 0 * NaN from them.  A key
  // past f16's range is NaN too (minus infinity would drop its position; two parts, infinities of both signs, do not);
  // such a value stays infinite, and its 64 are marked.
  constexpr int RB = MP < 8 * NW ? MP / NW : 8;
  for (int r0 = wv; r0 < MP; r0 += NW * RB) {
    float v[RB][WIDE ? 8 : 1];
    h8_t hv[RB];
    const int k = 8 * lane;
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const int64_t at = s_row[r0 + NW * i];
      const bool on = at >= 0 && k < c.rank;
      if constexpr (WIDE) {
        if (on) load8<float>(rows + at + k, v[i]);
        else
#pragma unroll
          for (int e = 0; e < 8; e++) v[i][e] = 0.f;
      } else {
        const h8_t z = {};
        hv[i] = on ? *reinterpret_cast<const h8_t*>(rows + at + k) : z;
      }
    }
#pragma unroll
    for (int i = 0; i < RB; i++) {
      if constexpr (WIDE) {
        h8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          _Float16 p, q;
          split2(v[i][e], p, q);
          hi[e] = p, lo[e] = q;
        }
        *reinterpret_cast<h8_t*>(&s_c[0][r0 + NW * i][k]) = hi;
        *reinterpret_cast<h8_t*>(&s_c[CP - 1][r0 + NW * i][k]) = lo;
        hv[i] = hi;
      } else {
        *reinterpret_cast<h8_t*>(&s_c[0][r0 + NW * i][k]) = hv[i];
      }
      typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
      float odd = 0.f;  // sum of 0 * value
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        odd = __builtin_amdgcn_fdot2(h2_t{hv[i][e], hv[i][e + 1]}, h2_t{_Float16(0), _Float16(0)}, odd, false);
      if (__ballot(odd != 0.f) && lane == 0) s_row[r0 + NW * i] = -3;
    }
  }
  __syncthreads();

  for (; w0 < w_end; w0 += STEP) {
    f4_t acc[4][MJ];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < MJ; j++) acc[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < pairs; p0 += 2) {
#pragma unroll
      for (int pp = 0; pp < 2; pp++) {
        const int p = p0 + pp;
        if (p >= pairs) break;
        if (p + 1 < pairs) read_w(p + 1, a[pp ^ 1]);
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
          for (int q = 0; q < CP; q++)
#pragma unroll
            for (int j0 = 0; j0 < MJ; j0 += JB) {  // 4 operands at a time: registers
              h8_t b[JB];
#pragma unroll
              for (int j = 0; j < JB; j++)
                b[j] = *reinterpret_cast<const h8_t*>(&s_c[q][16 * (j0 + j) + col][64 * p + 16 * g + 8 * s]);
#pragma unroll
              for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < JB; j++) acc[i][j0 + j] = mfma(a[pp][i][s], b[j], acc[i][j0 + j]);
            }
      }
    }
    const int h = w0 / WP, n0 = w0 % WP;
    rows_of(w0 + STEP);  // the next rows' first operands are on their way during the stores
    if (w0 + STEP < w_end) read_w(0, a[0]);
    const bool key = n0 < NT;
    _Float16* const dst = key ? x.k : x.v;
    const int64_t plane = key ? x.k_plane : x.v_plane;
    const int width = key ? NT : VT, n = (key ? n0 : n0 - NT) + 16 * g;
#pragma unroll
    for (int j = 0; j < MJ; j++) {
      const int64_t row = s_row[16 * j + col];
      if (row == -2) continue;
      const bool odd = row == -3;
      const float instead = key ? NAN : 0.f;
      if (!key) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(acc[e / 4][j][e % 4]));
        const uint64_t past = __ballot(!odd && !(top < 65520.f));
        if (g == 0)
          x.odd[(int64_t(h) * x.total + m0 + 16 * j + col) * (VT / 64) + (n0 - NT) / 64] =
              ((past >> col) & 0x0001000100010001ull) != 0;
      }
      _Float16* p = dst + (int64_t(h) * x.total + m0 + 16 * j + col) * width + n;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        h8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          _Float16 y, z;
          const float sum = acc[2 * half + e / 4][j][e % 4];
          split2(odd || (!TWO && key && !(fabsf(sum) < 65520.f)) ? instead : sum, y, z);
          hi[e] = y, lo[e] = z;
        }
        *reinterpret_cast<h8_t*>(p + 8 * half) = hi;
        if (TWO) *reinterpret_cast<h8_t*>(p + plane + 8 * half) = lo;
      }
    }
  }
}

constexpr int kFlashRows = 128;  // tokens a workgroup: 32 a wave

// Shape of the attention kernel: KR positions a step, in LDS as rows of keys, key parts and values (and of their
// lower parts), chunks swapped by the row's number; two such buffers, two workgroups a CU.
template <int NT, int PT, int VT, bool TWO>
struct FlashShape {
  static constexpr int kPlanes = TWO ? 2 : 1;
  // (64 positions where two workgroups' LDS holds them: 901 us for 4097 f16 tokens of 128 heads, by 32s 952)
  static constexpr int KR = NT + PT + VT <= 320 && !TWO ? 64 : 32;
  static constexpr int kKey = KR * NT * 2, kRope = KR * PT * 2, kVal = KR * VT * 2;
  static constexpr int kPlane = kKey + kRope + kVal;
  static constexpr int kBuf = kPlane * kPlanes;
  // workgroups a CU: as LDS allows, and the registers of 32 tokens' accumulators
  static constexpr int kGroups = 4 * kBuf <= 160 * 1024 && VT <= 128 ? 2 : 1;
  static_assert(2 * kBuf <= 160 * 1024 && kKey % 4096 == 0 && kRope % 1024 == 0 && kVal % 4096 == 0, "tile shape");
};

// What a block of the attention works on: tile of the nh heads' tiles.
struct FlashTile {
  int h, seq, first, count, len, steps;  // head, sequence, token rows, the sequence's positions, steps of kr
  int64_t base, shift;                   // its first expanded row; the position of token row t is shift + t
};
__device__ __forceinline__ bool flash_tile(const LatentCache& c, int64_t total, int nh, int tiles, int kr, int lane,
                                           FlashTile& f) {
  // a head's blocks on one XCD (blocks go round the 8), so that its keys and values stay in one L2
  int k;
  if (nh % 8 == 0) {
    const int slot = blockIdx.x >> 3, per = nh / 8;
    f.h = (slot % per) * 8 + (blockIdx.x & 7);
    k = slot / per;
  } else {
    f.h = blockIdx.x % nh;
    k = blockIdx.x / nh;
  }
  // The late tiles, which attend to the most, first; where all blocks run at once, two a CU, the second half
  // of them in rising order, so that a CU gets a late tile and an early one.
  const int half = (tiles + 1) / 2;
  const int tile = tiles * nh <= 2 * 256 + nh && k >= half ? k - half : tiles - 1 - k;
  // tiles of 128 tokens, sequence after sequence
  int before = 0, end = 0;
  f.seq = -1;
  mla_sequences(c, total, lane, [&](int s, int64_t b, int n) {
    int s0 = s, s1 = s + 1;
    if (c.starts) s0 = c.starts[s], s1 = c.starts[s + 1];
    const int from = max(s0, 0), mine = max(min(s1, c.n_tokens) - from, 0), nt = (mine + kFlashRows - 1) / kFlashRows;
    if (tile < before + nt) {
      f.seq = s, f.first = from + (tile - before) * kFlashRows;
      f.count = min(kFlashRows, mine - (tile - before) * kFlashRows);
      f.base = b, f.len = n, end = s1;
      return false;
    }
    before += nt;
    return true;
  });
  if (f.seq < 0) return false;
  f.shift = int64_t(c.lens[f.seq]) - end;
  const int top = int(max(int64_t(0), min(f.shift + f.first + f.count, int64_t(f.len))));
  f.steps = (top + kr - 1) / kr;
  return true;
}

// Causal attention of 128 tokens of a sequence and a head, one pass with a running maximum and sum.  S^T =
// K q^T (positions x tokens) leaves a token per lane column and, taken in the order 4g .. 4g + 3, 16 + 4g .. of
// 32 positions, is the B operand of O^T += V^T p, V^T read from LDS transposed: numerators, factors and
// accumulators of a token stay in its lanes.  Accumulators are rescaled only where a maximum grew by 2^kFlashGrow.
// f16 activations: queries, keys, values and numerators are one part, and an output is off by 0.0004 of its size, its
// own rounding 0.0002; as two parts (f32 activations have them) 4097 tokens of 128 heads take 2.3 ms in all against 1.1.
// Grid y: runs of `cut` steps; a tile of more than one leaves a partial row a token and run (part_o, part_ml),
// which mla_flash_merge_kernel joins.
//
// Measured: 4097 tokens of 128 heads of 192 and 128 (f16): 850 to 900 us, 760 to 810 TFLOP/s of what the mask leaves;
// 2048 tokens of 32 heads with two-part products (three for each): 162 us, 800 TFLOP/s of products.  Bound by the products and, half
// as long, the softmax between them: 32 tokens a wave and two workgroups a CU let one's products run under the
// other's softmax.
template <int NT, int PT, int VT, typename X, bool TWO>
__global__ void __launch_bounds__(256, (FlashShape<NT, PT, VT, TWO>::kGroups))
    mla_flash_kernel(LatentCache c, const X* __restrict__ q, int64_t q_stride, int nope, int v_dim, int nh, int h0,
                     Expanded x, float scale, MlaRope rope, X* __restrict__ out, int64_t out_stride, int tiles, int cut,
                     float* __restrict__ part_o, float2* __restrict__ part_ml) {
  using S = FlashShape<NT, PT, VT, TWO>;
  constexpr int KR = S::KR, RT = KR / 16, KT = (NT + PT) / 32, DT = VT / 16;
  __shared__ __attribute__((aligned(16))) uint8_t s_kv[2 * S::kBuf];
  const uint32_t lds0 = uint32_t(uintptr_t((lds_u8*)s_kv));
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  FlashTile ft;
  if (!flash_tile(c, x.total, nh, tiles, KR, lane, ft)) return;
  const int h = ft.h, seq = ft.seq, first = ft.first, count = ft.count, len = ft.len;
  const int64_t base = ft.base, shift = ft.shift;
  const int units = (ft.steps + cut - 1) / cut;
  const int begin = int(blockIdx.y) * cut, steps = min(ft.steps, begin + cut);
  if (blockIdx.y > 0 && int(blockIdx.y) >= units) return;

  // the queries: B operands, each token's brought near 1 by a power of two that goes into the scores' factor
  h8_t qh[2][KT], ql[2][TWO ? KT : 1];
  float factor[2];
  int limit[2];  // positions the lane's tokens attend to
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int i = wv * 32 + 16 * j + col;
    const int t = first + min(i, count - 1);
    const int64_t pos = shift + t;
    limit[j] = i < count ? int(max(int64_t(0), min(pos + 1, int64_t(len)))) : 0;
    const X* qr = q + t * q_stride + int64_t(h0 + h) * (nope + c.rope);
    float v[KT][8], mx = 0.f;
#pragma unroll
    for (int k = 0; k < KT; k++) {
      const int d = 32 * k + 8 * g;
      const bool on = d < NT ? d < nope : d - NT < c.rope;
      load8<X>(qr + (on ? (d < NT ? d : nope + d - NT) : 0), v[k]);
      if (d >= NT && rope.on) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 cs = mla_cos_sin(rope, on ? (d - NT + e) / 2 : 0, int(pos));
          const float a = v[k][e], b = v[k][e + 1];
          v[k][e] = a * cs.x - b * cs.y;
          v[k][e + 1] = a * cs.y + b * cs.x;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        v[k][e] = on ? v[k][e] : 0.f;
        mx = fmaxf(mx, fabsf(v[k][e]));
      }
    }
    mx = max_over_groups(mx);
    int ex = 0;
    if (mx > 0.f && mx < INFINITY) ex = ilogbf(mx);
    factor[j] = ldexpf(fabsf(scale) * 1.44269504088896341f, ex);  // its sign goes into the queries
#pragma unroll
    for (int k = 0; k < KT; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        _Float16 a, b;
        split2(ldexpf(scale < 0.f ? -v[k][e] : v[k][e], -ex), a, b);
        qh[j][k][e] = a;
        if (TWO) ql[j][k][e] = b;
      }
  }
  // positions below the wave's first token's need no mask
  const int low = int(max(int64_t(0), min(shift + first + wv * 32 + 1, int64_t(len))));
  // below the first token's, all tokens of the block attend to a position
  const int common = int(max(int64_t(0), min(shift + first + 1, int64_t(len))));
  const int32_t* table = c.table + seq * c.table_stride;

  const uint8_t* const kb = reinterpret_cast<const uint8_t*>(x.k + (int64_t(h) * x.total + base) * NT);
  const uint8_t* const vb = reinterpret_cast<const uint8_t*>(x.v + (int64_t(h) * x.total + base) * VT);
  const uint8_t* const pb = reinterpret_cast<const uint8_t*>(x.p + base * PT);
  // Load i of 1024 bytes of a part with rows of 2 w bytes, into LDS from `to` on: the lane's row, and its byte in
  // the row (chunks swapped).  Steps that end behind the last position repeat it (and mask it).
  auto part = [&](int i, int p0, bool whole, const uint8_t* src, int w, bool four, uint32_t to) {
    const int b = i * 1024 + 16 * lane, r = b / (2 * w);
    const uint32_t in = uint32_t((b % (2 * w)) ^ (16 * (four ? swap4(r) : swap8(r))));
    if (whole) dma_row(src + int64_t(p0) * (2 * w), uint32_t(r * 2 * w) + in, to + i * 1024);
    else dma_row(src, uint32_t(min(p0 + r, len - 1)) * uint32_t(2 * w) + in, to + i * 1024);
  };
  auto load = [&](int step, int buf) {
    const int p0 = step * KR;
    auto all = [&](bool whole) {
#pragma unroll
      for (int pl = 0; pl < S::kPlanes; pl++) {
        const uint32_t to = lds0 + buf * S::kBuf + pl * S::kPlane;
        constexpr int NK = S::kKey / 1024, NR = S::kRope / 1024, NV = S::kVal / 1024;
#pragma unroll
        for (int i = 0; i < NK; i += 4) part(i + wv, p0, whole, kb + pl * x.k_plane * 2, NT, false, to);
#pragma unroll
        for (int i = 0; i < NR; i += 4)
          if (NR % 4 == 0 || i + wv < NR) part(i + wv, p0, whole, pb + pl * x.p_plane * 2, PT, PT == 32, to + S::kKey);
#pragma unroll
        for (int i = 0; i < NV; i += 4)
          part(i + wv, p0, whole, vb + pl * x.v_plane * 2, VT, false, to + S::kKey + S::kRope);
      }
    };
    if (p0 + KR <= len) all(true);
    else all(false);
  };
  // the block of a step's position lane, and whether its values are marked
  const uint8_t* const ob = x.odd + (int64_t(h) * x.total + base) * (VT / 64);
  uint32_t ids = 0, marks = 0;
  auto find = [&](int step) {
    typedef std::conditional_t<VT == 64, uint8_t, std::conditional_t<VT == 128, uint16_t, uint32_t>> mark_t;
    const int p = min(step * KR + (lane & (KR - 1)), len - 1);
    ids = uint32_t(table[p >> c.shift]);
    marks = reinterpret_cast<const mark_t*>(ob)[p];
  };

  f4_t o[2][DT];
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int d = 0; d < DT; d++) o[j][d] = f4_t{0.f, 0.f, 0.f, 0.f};
  float m[2] = {-INFINITY, -INFINITY};
  f4_t l[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};  // (4 times the same)
  const int kat = 16 * (g ^ swap8(col)), kat4 = 16 * ((4 + g) ^ swap8(col));
  const int rat = 16 * (PT == 64 ? g ^ swap8(col) : g ^ swap4(col)), rat4 = 16 * ((4 + g) ^ swap8(col));
  const int vr = 4 * g + (col >> 2);
  int vat[4];
#pragma unroll
  for (int d = 0; d < 4; d++) vat[d] = vr * VT * 2 + 16 * ((2 * d + ((col & 3) >> 1)) ^ swap8(vr)) + 8 * (col & 1);

  if (steps > begin) load(begin, begin & 1);
  if (steps > begin) find(begin);
  for (int i = begin; i < steps; i++) {
    dma_wait<0>();
    const uint64_t ok = __ballot(ids < c.n_blocks);  // (their loads have come with the others: waited for before)
    const uint64_t odd = __ballot(marks != 0);
    __syncthreads();
    if (i + 1 < steps) {
      load(i + 1, (i + 1) & 1);
      find(i + 1);
    }
    const uint8_t* kv = s_kv + (i & 1) * S::kBuf;
    const int p0 = i * KR;
    // Rows of values past f16's range, of which a token that does not attend to them would take 0 * infinity, are made
    // zeros, and their key parts NaN.  (Looked for here, not marked when they were made: 1 to 2 % more.)
    if (odd && p0 + KR > common) {
      constexpr int L = VT / 8;  // lanes a row
      uint8_t* const rows = s_kv + (i & 1) * S::kBuf;
      uint32_t z1 = 0u, nan1 = 0x7E007E00u;
      int id = lane;
      asm volatile("" : "+v"(z1), "+v"(nan1), "+v"(id));  // (what hangs on these stays in here, out of the loop's registers)
      const u32x4 z = {z1, z1, z1, z1}, nan = {nan1, nan1, nan1, nan1};
      for (int r = wv; r < KR; r += 4)
        if ((odd >> r) & 1) {
          if (id < L * S::kPlanes)
            *reinterpret_cast<u32x4*>(rows + S::kKey + S::kRope + (id / L) * S::kPlane + r * VT * 2 + 16 * (id % L)) = z;
          if (id < PT / 8) *reinterpret_cast<u32x4*>(rows + S::kKey + r * PT * 2 + 16 * id) = nan;
        }
      __syncthreads();
    }
    f4_t s[2][RT];
    // operands are read a group of products ahead
    constexpr int KP = S::kPlanes;
    h8_t ka[2][RT][KP];
    auto read_k = [&](int k) {
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const int row = 16 * r + col;
        const uint8_t* p = k < NT / 32 ? kv + row * NT * 2 + ((k & 1) ? kat4 : kat) + 128 * (k >> 1)
                                       : kv + S::kKey + row * PT * 2 + (((k - NT / 32) & 1) ? rat4 : rat);
#pragma unroll
        for (int e = 0; e < KP; e++) ka[k & 1][r][e] = *reinterpret_cast<const h8_t*>(p + e * S::kPlane);
      }
    };
    read_k(0);
#pragma unroll
    for (int k = 0; k < KT; k++) {
      if (k + 1 < KT) read_k(k + 1);
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          s[j][r] = mfma(ka[k & 1][r][0], qh[j][k], k ? s[j][r] : f4_t{0.f, 0.f, 0.f, 0.f});
      if constexpr (TWO) {
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int j = 0; j < 2; j++) s[j][r] = mfma(ka[k & 1][r][0], ql[j][k], s[j][r]);
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int j = 0; j < 2; j++) s[j][r] = mfma(ka[k & 1][r][KP - 1], qh[j][k], s[j][r]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    h8_t bh[2][RT / 2], bl[2][RT / 2];
    bool grew[2];
    float alpha[2];
    const bool masked = p0 + KR > low || ok != ~0ull;
    float times[2] = {factor[0], factor[1]};
    if (masked) {
      const uint64_t mine = ok >> (4 * g);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        times[j] = 1.f;
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            s[j][r][e] = p0 + 16 * r + 4 * g + e < limit[j] && (mine & (1ull << (16 * r + e))) ? s[j][r][e] * factor[j]
                                                                                                : -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float mx = s[j][0][0];
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[j][r][e]);
      mx = max_over_groups(mx) * times[j];
      grew[j] = __any(mx > m[j] + kFlashGrow);
      const float mn = grew[j] ? fmaxf(m[j], mx) : m[j];
      const float ref = mn == -INFINITY ? 0.f : mn, from = ref - kFlashLift;
      alpha[j] = __builtin_amdgcn_exp2f(m[j] - ref);
      m[j] = mn;
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
    for (int j = 0; j < 2; j++)
      if (grew[j]) {
        l[j] *= alpha[j];
#pragma unroll
        for (int d = 0; d < DT; d++) o[j][d] *= alpha[j];
      }
    // the sums of the numerators, as the product rounds them: a row of ones in place of the values
    {
      h8_t one;
#pragma unroll
      for (int e = 0; e < 8; e++) one[e] = _Float16(1.f);
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int r = 0; r < RT / 2; r++) {
          l[j] = mfma(one, bh[j][r], l[j]);
          if constexpr (TWO) l[j] = mfma(one, bl[j][r], l[j]);
        }
    }
    const uint8_t* vp = kv + S::kKey + S::kRope;
    auto tr = [&](int d, int r, int plane) {
      return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s4*)(vp + plane * S::kPlane + vat[d & 3] + 128 * (d >> 2) + 16 * r * VT * 2));
    };
    h8_t va[2][RT / 2][KP];
    auto read_v = [&](int d) {
#pragma unroll
      for (int r = 0; r < RT / 2; r++)
#pragma unroll
        for (int e = 0; e < KP; e++)
          va[d & 1][r][e] = __builtin_bit_cast(
              h8_t, __builtin_shufflevector(tr(d, 2 * r, e), tr(d, 2 * r + 1, e), 0, 1, 2, 3, 4, 5, 6, 7));
    };
    read_v(0);
#pragma unroll
    for (int d = 0; d < DT; d++) {
      if (d + 1 < DT) read_v(d + 1);
#pragma unroll
      for (int r = 0; r < RT / 2; r++) {
#pragma unroll
        for (int j = 0; j < 2; j++) o[j][d] = mfma(va[d & 1][r][0], bh[j][r], o[j][d]);
        if constexpr (TWO) {
#pragma unroll
          for (int j = 0; j < 2; j++) o[j][d] = mfma(va[d & 1][r][0], bl[j][r], o[j][d]);
#pragma unroll
          for (int j = 0; j < 2; j++) o[j][d] = mfma(va[d & 1][r][KP - 1], bh[j][r], o[j][d]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const float sum = l[j][0];
    const int i = wv * 32 + 16 * j + col;
    if (i >= count) continue;
    if (units > 1) {
      const int64_t row = (int64_t(blockIdx.x) * gridDim.y + blockIdx.y) * kFlashRows + i;
#pragma unroll
      for (int d = 0; d < DT; d++) *reinterpret_cast<f4_t*>(part_o + row * VT + 16 * d + 4 * g) = o[j][d];
      if (g == 0) part_ml[row] = make_float2(m[j], sum);
      continue;
    }
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    X* dst = out + (first + i) * out_stride + int64_t(h0 + h) * v_dim;
#pragma unroll
    for (int d = 0; d < DT; d++) {
      const int v = 16 * d + 4 * g;
      if (v >= v_dim) continue;
      if constexpr (sizeof(X) == 4) {
        *reinterpret_cast<f4_t*>(dst + v) = o[j][d] * inv;
      } else {
        h4_t y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = _Float16(o[j][d][e] * inv);
        *reinterpret_cast<h4_t*>(dst + v) = y;
      }
    }
  }
}

// Joins the partial rows of a tile's runs: VT / 4 lanes a token.
template <int VT, typename X>
__global__ void __launch_bounds__(256) mla_flash_merge_kernel(LatentCache c, int64_t total, int v_dim, int nh, int h0, int kr,
                                                              X* __restrict__ out, int64_t out_stride, int tiles, int cut,
                                                              int runs, const float* __restrict__ part_o,
                                                              const float2* __restrict__ part_ml) {
  FlashTile f;
  if (!flash_tile(c, total, nh, tiles, kr, threadIdx.x & 63, f)) return;
  const int units = (f.steps + cut - 1) / cut;
  if (units <= 1) return;
  constexpr int L = VT / 4;
  const int v = 4 * (threadIdx.x % L);
  for (int i = blockIdx.y * (256 / L) + threadIdx.x / L; i < f.count; i += gridDim.y * (256 / L)) {
    const int64_t row = int64_t(blockIdx.x) * runs * kFlashRows + i;
    float m = -INFINITY, sum = 0.f;
    for (int u = 0; u < units; u++) m = fmaxf(m, part_ml[row + int64_t(u) * kFlashRows].x);
    const float ref = m == -INFINITY ? 0.f : m;
    f4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int u = 0; u < units; u++) {
      const int64_t at = row + int64_t(u) * kFlashRows;
      const float2 ml = part_ml[at];
      const float e = __builtin_amdgcn_exp2f(ml.x - ref);
      sum += e * ml.y;
      acc += e * *reinterpret_cast<const f4_t*>(part_o + at * VT + v);
    }
    if (v >= v_dim) continue;
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    X* dst = out + (f.first + i) * out_stride + int64_t(h0 + f.h) * v_dim + v;
#pragma unroll
    for (int e = 0; e < 4; e++) dst[e] = X(acc[e] * inv);
  }
}

// ---------------------------------------------------------------- host

// The padded widths that a head's take: the smallest of the three the kernels are built for.
struct PrefillShape {
  int nt, pt, vt;
};
static PrefillShape prefill_shape(int nope, int rope, int v) {
  if (nope <= 64 && rope <= 32 && v <= 64) return {64, 32, 64};
  if (nope <= 128 && v <= 128) return {128, 64, 128};
  return {256, 64, 256};
}

static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }
static size_t prefill_bytes(const PrefillShape& s, int64_t total, size_t heads, int planes) {
  return up256(size_t(total) * s.pt * 2 * planes) + up256(heads * size_t(total) * s.nt * 2 * planes) +
         up256(heads * size_t(total) * s.vt * 2 * planes) + up256(heads * size_t(total) * (s.vt / 64));
}

// Tiles of a call: a sequence's last may be short, so no more than this.
static int prefill_tiles(const LatentCache& c) {
  return c.starts ? c.n_tokens / kFlashRows + (c.n_seqs < c.n_tokens ? c.n_seqs : c.n_tokens) : c.n_seqs;
}

// Runs a tile's positions are cut into.  With fewer blocks than two a CU, cut so that about kFlashUnits
// runs come out, none below kFlashLeast positions; the partial rows of at most kFlashParts blocks x runs.  Six chunks of
// 17 to 600 tokens at the end of up to 2100 positions, 20 heads: 125 to 140 us and 13 for the merge, uncut 181; a
// prompt of 500, 20 heads: 28 and 6, uncut 40 (runs of 512 the same as uncut, of 192 25 and 7; a prompt of 700 32 and 8,
// by 512s 42 and 6, by 192s 34 and 9).
constexpr int kFlashUnits = 768, kFlashLeast = 256, kFlashParts = 1280;
struct FlashCut {
  int positions, runs;  // a run's positions, the most runs a tile has
};
static FlashCut flash_cut(int64_t blocks, int max_len) {
  FlashCut f{INT32_MAX / 2, 1};
  if (blocks >= 2 * 256) return f;
  int64_t p = (int64_t(max_len) * blocks + kFlashUnits - 1) / kFlashUnits;
  p = (p < kFlashLeast ? kFlashLeast : p + 63) / 64 * 64;
  const int64_t runs = (max_len + p - 1) / p;
  if (runs < 2 || runs * blocks > kFlashParts) return f;
  return {int(p), int(runs)};
}
static size_t flash_part_bytes(int vt) { return size_t(kFlashParts) * kFlashRows * (size_t(vt) * 4 + 8); }

template <int NT, int PT, int VT, typename X, typename KV, bool TWO>
static int launch_prefill(const LatentCache& c, const X* q, int64_t q_stride, int nh, int h0, int nope, int v_dim,
                          const _Float16* w, const Expanded& x, float scale, const MlaRope& rope, X* out,
                          int64_t out_stride, void* parts, hipStream_t s) {
  // Where 512 weight rows and the larger tile of positions a block leave more than half the CUs without one: 128 rows
  // and 32 positions a block.  A CU takes as long to draw 512 rows from memory whatever the positions: 23 positions of
  // 20 heads 11 us, with the larger blocks 21; 250 15 and 28; 500 19 and 30; 700 23 and 28.  With 400 positions of 128
  // heads, blocks for 192 CUs, 32 positions a block would read the weights twelve times (69 us and 32).
  // Otherwise weight rows a block: 512s, so that the rounds of one block a CU, each its 512s and what loading the
  // latents takes (about half of one), come out shortest.
  using S = ExpandShape<KV>;
  const int rows = nh * (NT + VT), all = (rows + 511) / 512;
  int64_t across = (x.total + S::kPos - 1) / S::kPos;
  if (across * all < 128) {
    across = (x.total + S::kShort - 1) / S::kShort;
    const dim3 ge(unsigned((rows + 127) / 128 + 1) * unsigned(across));
    hipLaunchKernelGGL((mla_expand_kernel<NT, PT, VT, KV, TWO, S::kShort, 2>), ge, dim3(128), 0, s, c, nh, nope, v_dim, w,
                       x, 128);
  } else {
    int run = all;
    double best = 0;
    for (int n = 1; n <= all; n++) {
      const int each = (all + n - 1) / n;
      const double cost = double((across * ((all + each - 1) / each) + 255) / 256) * (each + 0.5);
      if (n == 1 || cost < best) best = cost, run = each;
    }
    const dim3 ge(unsigned((all + run - 1) / run + 1) * unsigned(across));
    hipLaunchKernelGGL((mla_expand_kernel<NT, PT, VT, KV, TWO, S::kPos, 8>), ge, dim3(512), 0, s, c, nh, nope, v_dim, w,
                       x, run * 512);
  }
  int rc = check_launch("mla expand");
  if (rc) return rc;
  constexpr int KR = FlashShape<NT, PT, VT, TWO>::KR;
  const int tiles = prefill_tiles(c);
  const unsigned blocks = unsigned(tiles) * nh;
  const int longest = int(x.total < c.max_len ? x.total : c.max_len);
  const FlashCut f = parts ? flash_cut(blocks, longest) : FlashCut{INT32_MAX / 2, 1};
  float* part_o = static_cast<float*>(parts);
  float2* part_ml = reinterpret_cast<float2*>(part_o + size_t(kFlashParts) * kFlashRows * VT);
  hipLaunchKernelGGL((mla_flash_kernel<NT, PT, VT, X, TWO>), dim3(blocks, unsigned(f.runs)), dim3(256), 0, s, c, q,
                     q_stride, nope, v_dim, nh, h0, x, scale, rope, out, out_stride, tiles, f.positions / KR, part_o,
                     part_ml);
  if ((rc = check_launch("mla flash")) || f.runs == 1) return rc;
  hipLaunchKernelGGL((mla_flash_merge_kernel<VT, X>), dim3(blocks, 8), dim3(256), 0, s, c, x.total, v_dim, nh, h0, KR, out,
                     out_stride, tiles, f.positions / KR, f.runs, part_o, part_ml);
  return check_launch("mla flash merge");
}

}  // namespace jero

using namespace jero;

extern "C" size_t jero_hip_mla_prefill_workspace_bytes(const jero_latent_cache* cache, int act_dtype, int n_heads,
                                                       int nope_dim, int v_dim, int64_t total_len) {
  if (!cache || n_heads < 0 || nope_dim < 1 || v_dim < 1 || total_len < 1) return 0;
  const PrefillShape s = prefill_shape(nope_dim, cache->rope_dim, v_dim);
  const int planes = act_dtype == JERO_F16 ? 1 : 2;
  const size_t one = prefill_bytes(s, total_len, 1, planes), head = size_t(total_len) * ((s.nt + s.vt) * 2 * planes + s.vt / 64);
  if (n_heads == 0) return one;
  size_t heads = 1;
  if (one < (size_t(1) << 30)) heads += ((size_t(1) << 30) - one) / (head + 768);
  // (a call whose positions may be cut into runs, with room for their partial rows)
  const int64_t longest = total_len < cache->max_len ? total_len : cache->max_len;
  return prefill_bytes(s, total_len, heads < size_t(n_heads) ? heads : size_t(n_heads), planes) +
         (longest > kFlashLeast ? flash_part_bytes(s.vt) : 0);
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
  if (cache->n_seqs > kPrefillSeqs)
    return fail(JERO_ERR_CAPABILITY_MISMATCH, "mla_prefill_attention: more than " + std::to_string(kPrefillSeqs) + " sequences");
  if (total_len < 1 || total_len > (int64_t(1) << 23))
    return fail(JERO_ERR_TENSOR_BOUNDS, "mla_prefill_attention: total_len must be 1 to 2^23");
  MlaRope rope;
  if ((rc = mla_rope_of(rope_theta, cache->rope_dim, &rope))) return rc;
  const PrefillShape shape = prefill_shape(nope_dim, cache->rope_dim, v_dim);
  const int planes = act_dtype == JERO_F16 ? 1 : 2;
  void* ws = workspace_dev;
  if (!ws) {
    workspace_bytes = jero_hip_mla_prefill_workspace_bytes(cache, act_dtype, n_heads, nope_dim, v_dim, total_len);
    if ((rc = workspace(workspace_bytes, &ws))) return rc;
  }
  const size_t one = prefill_bytes(shape, total_len, 1, planes);
  if (workspace_bytes < one)
    return fail(JERO_ERR_TENSOR_BOUNDS, "mla_prefill_attention: workspace of " + std::to_string(workspace_bytes) +
                                            " bytes, need " + std::to_string(one));
  if (reinterpret_cast<uintptr_t>(ws) & 255u)
    return fail(JERO_ERR_INVALID_ARGUMENT, "mla_prefill_attention: workspace must be 256-byte aligned");
  const LatentCache c = mla_cache_of(cache, n_tokens);
  auto heads_in = [&](size_t bytes) {
    int n = n_heads;
    while (n > 1 && prefill_bytes(shape, total_len, size_t(n), planes) > bytes) n--;
    return n;
  };
  // heads at a time: those that fit beside the partial rows where such a call is cut into runs, else all that fit
  const size_t part_bytes = flash_part_bytes(shape.vt);
  const int longest = int(total_len < cache->max_len ? total_len : cache->max_len);
  int per = heads_in(workspace_bytes >= one + part_bytes ? workspace_bytes - part_bytes : workspace_bytes);
  if (flash_cut(int64_t(prefill_tiles(c)) * per, longest).runs == 1) per = heads_in(workspace_bytes);
  const size_t rows_bytes = prefill_bytes(shape, total_len, size_t(per), planes);
  void* const parts = workspace_bytes - rows_bytes >= part_bytes ? static_cast<uint8_t*>(ws) + rows_bytes : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int wide = nope_dim + v_dim;
  for (int h0 = 0; h0 < n_heads; h0 += per) {
    const int nh = n_heads - h0 < per ? n_heads - h0 : per;
    const _Float16* w = static_cast<const _Float16*>(kv_b_dev) + int64_t(h0) * wide * c.rank;
    Expanded x;
    uint8_t* at = static_cast<uint8_t*>(ws);
    x.total = total_len;
    x.p_plane = total_len * shape.pt;
    x.k_plane = int64_t(per) * total_len * shape.nt;
    x.v_plane = int64_t(per) * total_len * shape.vt;
    x.p = reinterpret_cast<_Float16*>(at);
    at += up256(size_t(x.p_plane) * 2 * planes);
    x.k = reinterpret_cast<_Float16*>(at);
    at += up256(size_t(x.k_plane) * 2 * planes);
    x.v = reinterpret_cast<_Float16*>(at);
    x.odd = at + up256(size_t(x.v_plane) * 2 * planes);
#define JERO_PREFILL(NT, PT, VT, X, KV, TWO)                                                                      \
  rc = launch_prefill<NT, PT, VT, X, KV, TWO>(c, static_cast<const X*>(q_dev), q_stride, nh, h0, nope_dim, v_dim, w, x, \
                                              scale, rope, static_cast<X*>(out_dev), out_stride, parts, s)
#define JERO_PREFILL_TYPES(NT, PT, VT)                                                       \
  if (act_dtype == JERO_F16) JERO_PREFILL(NT, PT, VT, _Float16, _Float16, false);            \
  else if (cache->kv_dtype == JERO_KV_F16) JERO_PREFILL(NT, PT, VT, float, _Float16, true);  \
  else JERO_PREFILL(NT, PT, VT, float, float, true)
    if (shape.nt == 64) {
      JERO_PREFILL_TYPES(64, 32, 64);
    } else if (shape.nt == 128) {
      JERO_PREFILL_TYPES(128, 64, 128);
    } else {
      JERO_PREFILL_TYPES(256, 64, 256);
    }
#undef JERO_PREFILL_TYPES
#undef JERO_PREFILL
    if (rc) return rc;
  }
  return JERO_OK;
}
