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
  const int lane = threadIdx.x & 63, s = base + lane;
  const bool in = s < p.seqs;
  NewTokens r{0, 0, 0};
  if (!p.cu) return in ? new_tokens(p, s) : r;
  int32_t first = 0, bound = 0;
  if (in) {
    first = p.cu[s];
    bound = p.cu[s + 1];
    r = checked_tokens(p, first, bound, p.seq_lens[s]);
  }
  int32_t end = r.n ? bound : 0;
  if (!__ballot(bound < first || (r.n && first < reach))) {  // bounds that do not fall
    const uint64_t some = __ballot(r.n > 0);
    if (some) reach = __shfl(end, 63 - __builtin_clzll(some));
    return r;
  }
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

// By counted_tokens' rule, whatever the bounds are.
__device__ inline TokenAt locate_by_rule(const Paged& p, int32_t tok) {
  int32_t reach = 0;
  for (int32_t base = 0; base < p.seqs; base += 64) {
    const NewTokens r = counted_tokens(p, base, reach);
    const uint64_t holds = __ballot(r.n && r.first <= tok && tok < r.first + r.n);
    if (!holds) continue;
    const int l = __builtin_ctzll(holds);
    return token_at(base + l, NewTokens{__shfl(r.first, l), __shfl(r.n, l), __shfl(r.len, l)}, tok);
  }
  return TokenAt{0, -1};
}

__device__ inline TokenAt locate(const Paged& p, int32_t tok) {
  if (!p.cu) {
    const int32_t s = tok / p.even;
    return token_at(s, new_tokens(p, s), tok);
  }
  const int lane = threadIdx.x & 63;
  int32_t most = INT32_MIN;  // the lane's largest bound so far
  for (int32_t base = 0; base < p.seqs; base += 64) {
    const int32_t i = min(base + lane, p.seqs - 1), end = p.cu[i + 1];
    // Sequences up to the one that holds the token end at or before it.
    const uint64_t behind = __ballot(base + lane < p.seqs && end > tok);
    if (!behind) {
      most = max(most, end);
      continue;
    }
    const int l = __builtin_ctzll(behind);
    const int32_t first = __shfl(p.cu[i], l);
    const TokenAt at =
        token_at(base + l, checked_tokens(p, first, __shfl(end, l), __shfl(p.seq_lens[i], l)), tok);
    // It holds the token, and none before it reaches behind its first one.
    if (at.pos >= 0 && !__ballot(most > first || (lane < l && end > first))) return at;
    return locate_by_rule(p, tok);
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
