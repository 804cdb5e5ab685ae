// drafts.hip -- drafted tokens accepted or replaced by given random numbers.
#include "jero_common.h"
#include "runtime.h"

namespace jero {

// A drafted token stands where u q < p; the next is the first token whose running sum of weights passes u times their
// total, weights max(p - q, 0) or p.  Two launches: the sums of 2048 weights a workgroup, then the search, by chunks and
// within one; for small vocabularies one workgroup a sequence does both.  Only the row that a token is drawn from is read.
// Bound by its bytes and, before them, three latencies (starts, tokens, probabilities): 64 chats of up to four drafts over
// 151936 tokens, 78 MB: 17.7 + 6.2 us, 4.4 TB/s; one chat, 32000: 11.5 us.  Chunks of 1024, 4096 and 8192: 21, 17.5 and 22 us
// and 7, 7 and 13.  64-bit sums of 32-bit values: no order of theirs moves a border by more than 2^-47 of the total.
constexpr int kDraftChunk = 2048;  // of the vocabulary, a workgroup

// Where a sequence's next token is drawn from.
struct Verdict {
  int first, rows;
  int accepted;  // -1: the sequence was not granted its rows
  int row;       // of the target's probabilities; -1: no rows
  int less;      // the draft's row taken off, or -1
  int without;   // a token that gets no weight, or -1
};

struct Drafts {
  const float *target, *draft, *u, *u_last;
  const int32_t *tokens, *starts, *granted;
  int64_t target_stride, draft_stride;
  int n_tokens, n_drafts, vocab, chunks;
  int32_t *out, *accepted, *dropped;
  double* sums;       // [n_seqs][chunks]: of the weights
  Verdict* verdicts;  // [n_seqs]
};

// By a whole workgroup of whole waves; s_n: one int of LDS.  Each wave finds the same.
__device__ __forceinline__ Verdict verdict_of(const Drafts& d, int s, int* s_n) {
  const int tid = threadIdx.x, lane = tid & 63;
  Verdict v;
  v.first = min(max(d.starts[s], 0), d.n_tokens);
  v.rows = min(max(d.starts[s + 1], v.first), d.n_tokens) - v.first;
  v.accepted = d.granted && !d.granted[s] ? -1 : 0, v.row = v.less = v.without = -1;
  // The drafted tokens of the sequences before.  Each sum stops at all there are, behind which none is this sequence's:
  // whatever the starts are, it does not wrap (16 waves of at most 2^22).
  if (tid == 0) *s_n = 0;
  __syncthreads();
  int n = 0;
  auto start = [&](int i) { return min(max(d.starts[i], 0), d.n_tokens); };
  for (int i = tid; i < s; i += blockDim.x) n = min(n + max(start(i + 1) - start(i) - 1, 0), d.n_drafts);
  n = min(group_sum_i<64>(n), d.n_drafts);
  if (lane == 0 && n) atomicAdd(s_n, n);
  __syncthreads();
  const int before = *s_n;
  if (v.rows < 1 || v.accepted < 0) return v;
  const int drafted = max(min(v.rows - 1, d.n_drafts - before), 0);
  int at = drafted;  // the first that is refused
  for (int j0 = 0; j0 < drafted && at == drafted; j0 += kWave) {
    const int j = j0 + lane;
    bool good = true;
    if (j < drafted) {
      const int x = d.tokens[v.first + j + 1];
      good = false;
      if (x >= 0 && x < d.vocab) {
        const double p = d.target[(v.first + j) * d.target_stride + x];
        const double q = d.draft ? double(d.draft[(before + j) * d.draft_stride + x]) : 1.0;
        good = double(d.u[before + j]) * q < p;
      }
    }
    const uint64_t bad = __ballot(!good);
    if (bad) at = j0 + __builtin_ctzll(bad);
  }
  v.accepted = at;
  v.row = v.first + at;
  if (at < drafted) {
    if (d.draft) v.less = before + at;
    else v.without = d.tokens[v.row + 1];
  }
  return v;
}

__device__ __forceinline__ double finite_weight(double w) { return w > 0.0 && w < 1e300 ? w : 0.0; }

// The weight of token i: the target's probability less the draft's.
__device__ __forceinline__ double weight_of(const Verdict& v, const float* p, const float* q, int i) {
  const double w = p[i];
  if (q) return finite_weight(w - double(q[i]));
  return i == v.without ? 0.0 : finite_weight(w);
}

// The weights of tokens [lo, lo + 4 n), four a lane and step: all loads before the sum.
template <int N, typename L>
__device__ __forceinline__ double sum_weights(const Verdict& v, const float* p, const float* q, int lo, int step, L load) {
  float4 a[N], b[N];
#pragma unroll
  for (int n = 0; n < N; n++) a[n] = load(p + lo + n * step);
  if (q)
#pragma unroll
    for (int n = 0; n < N; n++) b[n] = load(q + lo + n * step);
  double sum = 0.0;
#pragma unroll
  for (int n = 0; n < N; n++) {
    const float x[4] = {a[n].x, a[n].y, a[n].z, a[n].w}, y[4] = {b[n].x, b[n].y, b[n].z, b[n].w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const double w = q ? double(x[e]) - double(y[e]) : double(x[e]);
      sum += lo + n * step + e == v.without ? 0.0 : finite_weight(w);
    }
  }
  return sum;
}

// The sum of a chunk's weights, by 256 threads; s: 4 of LDS.  Thread 0 has it.
__device__ __forceinline__ double chunk_sum(const Drafts& d, const Verdict& v, const float* p, const float* q, int chunk,
                                            double* s, int tid) {
  const int lo = chunk * kDraftChunk, hi = min(lo + kDraftChunk, d.vocab);
  double sum = 0.0;
  if (hi - lo == kDraftChunk) {
    constexpr int N = kDraftChunk / 1024;
    if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0) {
      sum = sum_weights<N>(v, p, q, lo + 4 * tid, 1024, [](const float* x) { return *reinterpret_cast<const float4*>(x); });
    } else {  // (rows of an odd vocabulary)
      sum = sum_weights<N>(v, p, q, lo + 4 * tid, 1024, [](const float* x) { return make_float4(x[0], x[1], x[2], x[3]); });
    }
  } else {
    for (int i = lo + tid; i < hi; i += 256) sum += weight_of(v, p, q, i);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  __syncthreads();
  if ((tid & 63) == 0) s[tid >> 6] = sum;
  __syncthreads();
  return s[0] + s[1] + s[2] + s[3];
}

// What is known of a sequence is written by one workgroup of it.  One that was not granted its rows holds none of their
// positions, so that none is to be taken back.
__device__ __forceinline__ void write_verdict(const Drafts& d, const Verdict& v, int s, int tid, int threads) {
  if (tid == 0) {
    d.accepted[s] = max(v.accepted, 0);
    if (d.dropped) d.dropped[s] = v.accepted < 0 ? 0 : max(v.rows - 1, 0) - v.accepted;
  }
  for (int i = tid; i < v.rows; i += threads)
    if (i != v.accepted) d.out[v.first + i] = i < v.accepted ? d.tokens[v.first + i + 1] : -1;
}

// The sums of a sequence's chunks by the waves of one workgroup, a chunk each.
__device__ __forceinline__ void wave_sums(const Drafts& d, const Verdict& v, const float* p, const float* q, double* sums,
                                          int tid, int waves) {
  for (int c = tid >> 6; c < d.chunks; c += waves) {
    double sum = 0.0;
    const int lo = c * kDraftChunk, hi = min(lo + kDraftChunk, d.vocab), lane = tid & 63;
    if (hi - lo == kDraftChunk && ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0)
      sum = sum_weights<kDraftChunk / 256>(v, p, q, lo + 4 * lane, 256,
                                           [](const float* x) { return *reinterpret_cast<const float4*>(x); });
    else
      for (int i = lo + lane; i < hi; i += kWave) sum += weight_of(v, p, q, i);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
    if ((tid & 63) == 0) sums[c] = sum;
  }
}

// Workgroup (chunk, sequence): the sum of its chunk's weights; the first chunk's writes what is known of the sequence.
__global__ void __launch_bounds__(256) draft_sums_kernel(Drafts d) {
  __shared__ int s_n;
  __shared__ double s_sum[4];
  const int s = blockIdx.y, tid = threadIdx.x;
  const Verdict v = verdict_of(d, s, &s_n);
  if (blockIdx.x == 0) {
    if (tid == 0) d.verdicts[s] = v;
    write_verdict(d, v, s, tid, 256);
  }
  if (v.row < 0) return;
  const double sum = chunk_sum(d, v, d.target + v.row * d.target_stride,
                               v.less >= 0 ? d.draft + v.less * d.draft_stride : nullptr, blockIdx.x, s_sum, tid);
  if (tid == 0) d.sums[int64_t(s) * d.chunks + blockIdx.x] = sum;
}

// Inclusive sums over the workgroup's 1024 threads; s: 16 of LDS.
__device__ __forceinline__ double scan1024(double v, double* s, int tid) {
  const int lane = tid & 63;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const double o = __shfl_up(v, off, kWave);
    if (lane >= off) v += o;
  }
  __syncthreads();
  if (lane == 63) s[tid >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 15; w++) {
    const double o = s[w];
    if (w < (tid >> 6)) v += o;
  }
  return v;
}

// The lowest of the workgroup's `at` and the highest of its `last` (both rise with the thread): one lane a wave asks, as
// 64 lanes' operations on one word go one after another.
__device__ __forceinline__ void lowest_and_highest(int at, int last, int* s_at, int* s_last, int lane) {
  const uint64_t found = __ballot(at != INT32_MAX), any = __ballot(last >= 0);
  if (found && lane == __builtin_ctzll(found)) atomicMin(s_at, at);
  if (any && lane == 63 - __builtin_clzll(any)) atomicMax(s_last, last);
}

// Workgroup a sequence: finds the chunk, then the token in it.  WHOLE: the sums are its own work too.
constexpr int kPickThreads = 1024, kPickChunks = (1 << 24) / kDraftChunk / kPickThreads;  // a thread, at most
constexpr int kWholeChunks = 32;
template <bool WHOLE>
__global__ void __launch_bounds__(kPickThreads) draft_pick_kernel(Drafts d) {
  __shared__ int s_at, s_last, s_n;
  __shared__ double s_scan[16], s_before, s_total, s_sums[WHOLE ? kWholeChunks : 1];
  const int s = blockIdx.x, tid = threadIdx.x;
  double* const sums = WHOLE ? s_sums : d.sums + int64_t(s) * d.chunks;
  const float u = d.u_last[s];
  Verdict v;
  if constexpr (WHOLE) {
    v = verdict_of(d, s, &s_n);
    write_verdict(d, v, s, tid, kPickThreads);
    if (v.row < 0) return;
    wave_sums(d, v, d.target + v.row * d.target_stride, v.less >= 0 ? d.draft + v.less * d.draft_stride : nullptr, s_sums, tid,
              kPickThreads / kWave);
    __syncthreads();
  } else {
    v = d.verdicts[s];
  }
  const int each = (d.chunks + kPickThreads - 1) / kPickThreads, c0 = tid * each;  // chunks of a thread
  double w[kPickChunks];
  auto read = [&]() {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPickChunks; i++) sum += w[i] = i < each && c0 + i < d.chunks ? sums[c0 + i] : 0.0;
    return sum;
  };
  double mine = read();  // (on their way with the verdict)
  if (v.row < 0) return;
  const float* p = d.target + v.row * d.target_stride;
  const float* q = v.less >= 0 ? d.draft + v.less * d.draft_stride : nullptr;
  if (tid == 0) s_at = INT32_MAX, s_last = -1;
  double run = scan1024(mine, s_scan, tid);
  if (tid == kPickThreads - 1) s_total = run;
  __syncthreads();
  if (!(s_total > 0.0) && (q || v.without >= 0)) {
    // the draft takes off all there is: the target's own sums
    q = nullptr, v.without = -1;
    wave_sums(d, v, p, nullptr, sums, tid, kPickThreads / kWave);
    __syncthreads();
    mine = read();
    run = scan1024(mine, s_scan, tid);
    if (tid == kPickThreads - 1) s_total = run;
    __syncthreads();
  }
  const double passes = double(u) * s_total;
  // the first chunk whose running sum passes, or the last of any weight
  run -= mine;
  double before[kPickChunks];
  int at = INT32_MAX, last = -1;
#pragma unroll
  for (int i = 0; i < kPickChunks; i++) {
    before[i] = run;
    run += w[i];
    if (w[i] > 0.0) {
      if (run > passes) at = min(at, c0 + i);
      last = c0 + i;
    }
  }
  lowest_and_highest(at, last, &s_at, &s_last, tid & 63);
  __syncthreads();
  const int chunk = s_at != INT32_MAX ? s_at : s_last;
#pragma unroll
  for (int i = 0; i < kPickChunks; i++)
    if (i < each && c0 + i == chunk) s_before = before[i];
  __syncthreads();
  int drawn = -1;
  if (chunk >= 0) {
    if (tid == 0) s_at = INT32_MAX, s_last = -1;
    constexpr int N = kDraftChunk / kPickThreads;
    const int lo = chunk * kDraftChunk + N * tid;
    double x[N], sum = 0.0;
#pragma unroll
    for (int e = 0; e < N; e++) sum += x[e] = lo + e < d.vocab ? weight_of(v, p, q, lo + e) : 0.0;
    run = scan1024(sum, s_scan, tid) - sum + s_before;
    at = INT32_MAX, last = -1;
#pragma unroll
    for (int e = 0; e < N; e++) {
      run += x[e];
      if (x[e] > 0.0) {
        if (run > passes) at = min(at, lo + e);
        last = lo + e;
      }
    }
    lowest_and_highest(at, last, &s_at, &s_last, tid & 63);
    __syncthreads();
    drawn = s_at != INT32_MAX ? s_at : s_last;
  }
  if (tid == 0) d.out[v.first + v.accepted] = drawn;
}

}  // namespace jero

using namespace jero;

extern "C" size_t jero_hip_verify_drafts_workspace_bytes(int64_t n_seqs, int64_t vocab) {
  if (n_seqs < 1 || n_seqs > 65535 || vocab < 1 || vocab > (1 << 24)) return 0;
  const size_t chunks = size_t((vocab + kDraftChunk - 1) / kDraftChunk);
  return chunks <= kWholeChunks ? 0 : size_t(n_seqs) * (chunks * sizeof(double) + sizeof(Verdict));
}

extern "C" int jero_hip_verify_drafts_granted(const float* target_dev, int64_t target_stride, const float* draft_dev,
                                              int64_t draft_stride, const int32_t* tokens_dev, const int32_t* starts_dev,
                                              const int32_t* granted_dev, const float* u_dev, const float* u_last_dev,
                                              int64_t n_seqs, int64_t n_tokens, int64_t n_drafts, int64_t vocab,
                                              int32_t* out_dev, int32_t* accepted_dev, int32_t* dropped_dev,
                                              void* workspace_dev, size_t workspace_bytes, void* stream) {
  auto bad = [](int status, const char* what) { return fail(status, std::string("verify_drafts: ") + what); };
  if (!target_dev || !tokens_dev || !starts_dev || !u_last_dev || !out_dev || !accepted_dev || (n_drafts > 0 && !u_dev))
    return bad(JERO_ERR_INVALID_ARGUMENT, "null pointer");
  for (const void* p : {static_cast<const void*>(target_dev), static_cast<const void*>(draft_dev),
                        static_cast<const void*>(tokens_dev), static_cast<const void*>(starts_dev),
                        static_cast<const void*>(granted_dev), static_cast<const void*>(u_dev),
                        static_cast<const void*>(u_last_dev), static_cast<const void*>(out_dev),
                        static_cast<const void*>(accepted_dev), static_cast<const void*>(dropped_dev)})
    if (!aligned4(p)) return bad(JERO_ERR_INVALID_ARGUMENT, "arrays must be 4-byte aligned");
  if (n_seqs < 1 || n_tokens < 1 || vocab < 1 || n_drafts < 0 || n_drafts >= n_tokens)
    return bad(JERO_ERR_TENSOR_BOUNDS, "no sequences, tokens or vocabulary, or as many drafts as tokens");
  if (n_seqs > 65535 || n_tokens > (1 << 22) || vocab > (1 << 24))
    return bad(JERO_ERR_TENSOR_BOUNDS, "more than 65535 sequences, 2^22 tokens or a vocabulary of 2^24");
  if (target_stride < vocab || (draft_dev && draft_stride < vocab))
    return bad(JERO_ERR_TENSOR_BOUNDS, "rows overlap: a stride is below the vocabulary");
  // One launch, and no workspace, where a workgroup's reading of a whole row takes no longer than a second launch.
  const int64_t chunks = (vocab + kDraftChunk - 1) / kDraftChunk;
  const bool whole = chunks <= kWholeChunks;
  const size_t need = jero_hip_verify_drafts_workspace_bytes(n_seqs, vocab);
  if (!whole && workspace_dev) {
    if (workspace_bytes < need) return bad(JERO_ERR_TENSOR_BOUNDS, "the workspace is too small");
    if (reinterpret_cast<uintptr_t>(workspace_dev) & 15u)
      return bad(JERO_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  }
  // A sequence's inputs are read by several workgroups and waves, with no order between them and what one of them writes.
  struct Array {
    const void* p;
    int64_t n;
  };
  const Array ins[] = {{tokens_dev, n_tokens}, {starts_dev, n_seqs + 1}, {granted_dev, n_seqs}, {u_dev, n_drafts},
                       {u_last_dev, n_seqs}},
              outs[] = {{out_dev, n_tokens}, {accepted_dev, n_seqs}, {dropped_dev, n_seqs}};
  for (const Array& o : outs)
    for (const Array& i : ins) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(o.p), b = reinterpret_cast<uintptr_t>(i.p);
      if (a && b && a < b + 4 * uintptr_t(i.n) && b < a + 4 * uintptr_t(o.n))
        return bad(JERO_ERR_INVALID_ARGUMENT, "an output overlaps an input");
    }
  if (!whole && !workspace_dev)
    if (int rc = workspace(need, &workspace_dev)) return rc;
  Drafts d{};
  d.target = target_dev, d.draft = draft_dev, d.u = u_dev, d.u_last = u_last_dev;
  d.tokens = tokens_dev, d.starts = starts_dev, d.granted = granted_dev;
  d.target_stride = target_stride, d.draft_stride = draft_stride;
  d.n_tokens = int(n_tokens), d.n_drafts = int(n_drafts), d.vocab = int(vocab);
  d.chunks = int(chunks);
  d.out = out_dev, d.accepted = accepted_dev, d.dropped = dropped_dev;
  d.sums = static_cast<double*>(workspace_dev);
  d.verdicts = reinterpret_cast<Verdict*>(d.sums + n_seqs * d.chunks);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (whole) {
    hipLaunchKernelGGL((draft_pick_kernel<true>), dim3(unsigned(n_seqs)), dim3(kPickThreads), 0, s, d);
    return check_launch("verify_drafts");
  }
  const dim3 grid = {unsigned(d.chunks), unsigned(n_seqs), 1};
  hipLaunchKernelGGL(draft_sums_kernel, grid, dim3(256), 0, s, d);
  if (int rc = check_launch("verify_drafts sums")) return rc;
  hipLaunchKernelGGL((draft_pick_kernel<false>), dim3(unsigned(n_seqs)), dim3(kPickThreads), 0, s, d);
  return check_launch("verify_drafts");
}

extern "C" int jero_hip_verify_drafts(const float* target_dev, int64_t target_stride, const float* draft_dev,
                                      int64_t draft_stride, const int32_t* tokens_dev, const int32_t* starts_dev,
                                      const float* u_dev, const float* u_last_dev, int64_t n_seqs, int64_t n_tokens,
                                      int64_t n_drafts, int64_t vocab, int32_t* out_dev, int32_t* accepted_dev,
                                      int32_t* dropped_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  return jero_hip_verify_drafts_granted(target_dev, target_stride, draft_dev, draft_stride, tokens_dev, starts_dev, nullptr,
                                        u_dev, u_last_dev, n_seqs, n_tokens, n_drafts, vocab, out_dev, accepted_dev,
                                        dropped_dev, workspace_dev, workspace_bytes, stream);
}
