// Attention of chunks of new tokens, block by block (paged_chunk.hip).
#pragma once

#include <type_traits>

#include "paged.h"

namespace moba {

struct ChunkArgs {
  Paged p;
  const void *q, *k, *v;
  const int32_t* block_idx;  // [tokens, h_q, slots]
  void* out;
  float* lse;
  int32_t* n_items;          // work items of the call
  int32_t* table;            // [parts, h_kv, width]
  int4* items;               // (sequence * h_kv + kv head, block, first entry's place, entries)
  int32_t* entries;          // indices into the slice's [tokens, h_q, slots]
  float2* part_ml;           // (m, l) per entry
  float* part_acc;           // [entries, D]
  int32_t t0, t1;            // tokens of this slice
  int h_q, h_kv, slots;
  int part, parts, max_items;
  float scale_log2;
};

// Tokens per slice and part, bounds, and the workspace's layout (offsets).
struct ChunkPlan {
  int64_t slice, part, parts, max_items;
  size_t table, items, entries, ml, acc, total;
};

bool chunk_takes(const moba_paged& c);
ChunkPlan chunk_plan(const moba_paged& c);
int chunk_attend(const moba_paged& c, const Paged& p, void* workspace, hipStream_t s);

}  // namespace moba
