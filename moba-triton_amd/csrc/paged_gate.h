// Which blocks new tokens attend to over a paged cache (paged_gate.hip).
#pragma once

#include "paged.h"

namespace moba {

size_t gate_workspace(const moba_paged& c);
// Writes c.block_idx; rows of no sequence only with `all_rows`.
int gate_run(const moba_paged& c, const Paged& p, void* workspace, bool all_rows, hipStream_t s);

// The part-th run of a sequence's new tokens, at most `size` of them, inside
// the tokens [t0, t1). Parts are counted 64 sequences at a time by a wave's
// lanes.
struct Part {
  int32_t seq, begin, end;  // tokens; seq -1: no such part
};

__device__ inline Part find_part(const Paged& p, int32_t t0, int32_t t1, int32_t size, int32_t part) {
  const int lane = threadIdx.x & 63;
  int32_t before = 0;
  for (int32_t base = 0; base < p.seqs; base += 64) {
    NewTokens r{0, 0, 0};
    if (base + lane < p.seqs) r = new_tokens(p, base + lane);
    const int32_t lo = max(r.first, t0), hi = min(r.first + r.n, t1);
    const int32_t mine = hi > lo ? (hi - lo + size - 1) / size : 0;
    int32_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t y = __shfl_up(upto, off);
      if (lane >= off) upto += y;
    }
    const uint64_t past = __ballot(before + upto > part);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int32_t skip = part - before - (__shfl(upto, l) - __shfl(mine, l));
      Part out;
      out.seq = base + l;
      out.begin = __shfl(lo, l) + skip * size;
      out.end = min(out.begin + size, __shfl(hi, l));
      return out;
    }
    before += __shfl(upto, 63);
  }
  return Part{-1, 0, 0};
}

}  // namespace moba
