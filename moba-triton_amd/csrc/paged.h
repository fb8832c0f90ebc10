// Sequences whose keys and values lie in the pages of a cache: addressing
// shared by the kernels that write and read them.
//
// A page holds one MoBA block of every kv head: K and V [pages, h_kv, block,
// D], so that a block of a head is one contiguous run, and the blocks'
// representatives kbar [pages, h_kv, D]. Row s of the block table lists the
// pages of sequence s in order; seq_lens[s] counts its tokens with the new
// ones, which are its last. The new tokens of all sequences are packed along
// one token axis by cu_seqlens (null: the same number for every sequence).
#pragma once

#include "common.h"

namespace moba {

struct Paged {
  const int32_t* table;     // [seqs, width]
  const int32_t* seq_lens;  // [seqs]
  const int32_t* cu;        // [seqs + 1], or null
  int32_t seqs, width, pages;
  int32_t tokens;           // rows of the token axis
  int32_t even;             // new tokens per sequence where cu is null
  int32_t block;
};

// New tokens [first, first + n) of sequence s, at positions len - n, ..; n is
// 0 where the values make no sense, so no caller's buffer leads a kernel out
// of the token axis.
struct NewTokens {
  int32_t first, n, len;
};

__device__ inline NewTokens checked_tokens(const Paged& p, int32_t first, int32_t end, int32_t len) {
  const bool ok = first >= 0 && end > first && end <= p.tokens && len >= end - first;
  return NewTokens{first, ok ? end - first : 0, len};
}

__device__ inline NewTokens new_tokens(const Paged& p, int32_t s) {
  const int32_t first = p.cu ? p.cu[s] : s * p.even;
  return checked_tokens(p, first, p.cu ? p.cu[s + 1] : first + p.even, p.seq_lens[s]);
}

// The same for the sequences base, base + 1, .. of a wave's lanes (n 0 past the
// last), one call after another from base 0 on: a sequence counts only where no
// earlier one that makes sense by itself reaches behind its first token, so
// that no token has two sequences and their tokens are at most p.tokens in all.
// `reach`: where the earlier ones end, 0 at first.
__device__ inline NewTokens counted_tokens(const Paged& p, int32_t base, int32_t& reach) {
  const int lane = threadIdx.x & 63;
  NewTokens r{0, 0, 0};
  if (base + lane < p.seqs) r = new_tokens(p, base + lane);
  if (!p.cu) return r;
  int32_t end = r.n ? r.first + r.n : 0;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int32_t y = __shfl_up(end, off);
    if (lane >= off) end = max(end, y);
  }
  const int32_t up = __shfl_up(end, 1), before = max(reach, lane ? up : 0);
  if (r.first < before) r.n = 0;
  reach = max(reach, __shfl(end, 63));
  return r;
}

// Sequence and position of token `tok`, the same in all lanes of the wave;
// position -1 where the token belongs to no sequence (rows behind the last
// one, inconsistent lengths). Every lane holds the numbers of one of 64
// sequences, so up to 64 sequences take one round of loads.
struct TokenAt {
  int32_t seq, pos;
};

__device__ inline TokenAt token_at(int32_t s, const NewTokens& r, int32_t tok) {
  const int32_t i = tok - r.first;
  return TokenAt{s, i >= 0 && i < r.n ? r.len - r.n + i : -1};
}

__device__ inline TokenAt locate(const Paged& p, int32_t tok) {
  if (!p.cu) {
    const int32_t s = tok / p.even;
    return token_at(s, new_tokens(p, s), tok);
  }
  const int lane = threadIdx.x & 63;
  int32_t reach = 0;
  for (int32_t base = 0; base < p.seqs; base += 64) {
    NewTokens r = new_tokens(p, min(base + lane, p.seqs - 1));
    if (base + lane >= p.seqs) r.n = 0;
    const int32_t end = r.n ? r.first + r.n : 0;
    const uint64_t holds = __ballot(r.first <= tok && tok < end);
    if (holds) {
      // As counted_tokens: the first one that holds the token or none, for it
      // reaches behind the first tokens of the others that do.
      const int l = __builtin_ctzll(holds);
      const int32_t first = __shfl(r.first, l);
      if (first < reach || __ballot(lane < l && end > first)) break;
      return token_at(base + l, NewTokens{first, __shfl(r.n, l), __shfl(r.len, l)}, tok);
    }
    if (base + 64 < p.seqs) {
      int32_t most = end;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) most = max(most, __shfl_xor(most, off));
      reach = max(reach, most);
    }
  }
  return TokenAt{0, -1};
}

// What an address that is the same in all lanes of a wave holds, written by an
// earlier kernel: a scalar load, which no wait for vector memory includes.
__device__ inline int32_t uniform_load(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

// Page of block `blk` of sequence s, or -1 where the table has none.
__device__ inline int32_t page_of(const Paged& p, int32_t s, int32_t blk) {
  if (blk >= p.width) return -1;
  const int32_t id = p.table[static_cast<int64_t>(s) * p.width + blk];
  return id >= 0 && id < p.pages ? id : -1;
}

// Checks a call's shape and fills `p` (paged_attn.hip).
int paged_of(const moba_paged* c, Paged* p);

}  // namespace moba
