// paged.h -- attention over a paged key/value cache: what its kernels and the entry point share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jero_common.h"

namespace jero {

// A jero_paged_cache and a call's rows as the kernels take them.
struct PagedCall {
  const void *k, *v;
  const int32_t *table, *lens, *starts, *shared;
  int64_t table_stride, q_stride, out_stride;
  uint32_t n_blocks;
  int n_seqs, n_tokens, max_len, shared_len, shared_blocks;
  int shift;  // log2 of the block size
  int heads, kv_heads, group, dim;
  float scale;
};

// How a call's work is cut.  Its two phases, the shared positions for the rows of all sequences and each sequence's
// own from own_lo on, are cut into tiles of rows and chunks of positions; each chunk of a row is a part, joined
// by paged_merge_kernel where there are more than one.
constexpr int kNarrowRows = 16;
struct PagedPlan {
  int pre_blocks, pre_tiles, pre_chunks, pre_len;
  int own_blocks, own_tiles, own_chunks, own_len, own_lo;
  int parts;
  int wide_rows;
  int pre_wide, own_wide;
};

int paged_attend_64(const PagedCall& c, const PagedPlan& p, bool x16, bool kv16, const void* q, void* out, float* part_o,
                    float2* part_ml, hipStream_t s);
int paged_attend_128(const PagedCall& c, const PagedPlan& p, bool x16, bool kv16, const void* q, void* out, float* part_o,
                     float2* part_ml, hipStream_t s);
int paged_attend_256(const PagedCall& c, const PagedPlan& p, bool x16, bool kv16, const void* q, void* out, float* part_o,
                     float2* part_ml, hipStream_t s);

}  // namespace jero
