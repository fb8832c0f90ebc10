// Which blocks new tokens attend to over a paged cache (paged_gate.hip).
#pragma once

#include "paged.h"

namespace moba {

struct GateArgs {
  Paged p;
  const void* q;      // [tokens, h_q, D]
  const void* kbar;   // [pages, h_kv, D]
  uint32_t* keys;     // scores: [slice tokens, h_q, width]
  uint32_t* norms;    // tiles: [seqs, h_kv, kNormParts] float bits
  int32_t* block_idx; // [tokens, h_q, slots]
  int32_t tok0, slice;  // tokens [tok0, tok0 + slice) of this launch
  int h_q, h_kv, slots, take, current;
  int tile_tokens;    // tiles: tokens per workgroup
};

size_t gate_workspace(const moba_paged& c);
// Writes c.block_idx; rows of no sequence only with `all_rows`.
int gate_run(const moba_paged& c, const Paged& p, void* workspace, bool all_rows, hipStream_t s);

// Whether attention can choose from the scores by itself (paged_attn.hip), and
// the scores of all tokens into `workspace`: uint32 [tokens, h_q, width].
bool scores_only(const moba_paged& c);
int gate_scores(const moba_paged& c, const Paged& p, void* workspace, hipStream_t s);

// A rounded score as an integer in the order of the scores, 0 for what never
// ranks (-inf, NaN). 16-bit types: the upper half of the word.
template <typename T>
__device__ inline uint32_t score_key(float rounded) {
  uint32_t u = f2u(rounded + 0.f);
  const bool ranks = rounded > -INFINITY;
  if constexpr (T::kHalf) u = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(rounded + 0.f))) << 16;
  uint32_t o = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  if constexpr (T::kWords == 1) o &= 0xffff0000u;
  return ranks ? o : 0u;
}

// A wave's best TM entries: (score, id) in one word, larger first, so that
// equal scores go to the lower id; 0 for none. Each lane fills its own list.
// 16-bit types take 32-bit words (ids below 2^16), float32 64-bit ones.
template <typename T, int TM>
struct WaveBest {
  using Word = typename T::Word;
  Word best[TM];
  __device__ void clear() {
#pragma unroll
    for (int i = 0; i < TM; ++i) best[i] = 0;
  }
  __device__ static Word word(uint32_t key, int32_t j) {
    if constexpr (sizeof(Word) == 4) return key ? key | (0xffffu - static_cast<uint32_t>(j)) : 0u;
    return key ? (static_cast<Word>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(j)) : 0;
  }
  __device__ static int32_t id(Word w) {
    if constexpr (sizeof(Word) == 4) return static_cast<int32_t>(0xffffu - (w & 0xffffu));
    return static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(w));
  }
  __device__ void add(Word x) {
    if (x > best[TM - 1]) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const Word hi = max(x, best[i]);
        x = min(x, best[i]);
        best[i] = hi;
      }
    }
  }
  // Keys first, first + step, .. below n of a row, eight in flight.
  __device__ void add_all(const uint32_t* keys, int32_t n, int32_t first, int32_t step) {
    for (int32_t j0 = first; j0 < n; j0 += 8 * step) {
      uint32_t k[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) k[u] = keys[min(j0 + u * step, n - 1)];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int32_t j = j0 + u * step;
        if (j < n) add(word(k[u], j));
      }
    }
  }
  // The lanes' lists meet in six exchanges. The larger of entry i and the
  // other list's entry TM - 1 - i: the best TM of both, in an order that log2
  // TM exchange stages sort.
  __device__ void meet() {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      Word other[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) other[i] = __shfl_xor(best[i], off);
#pragma unroll
      for (int i = 0; i < TM; ++i) best[i] = max(best[i], other[TM - 1 - i]);
#pragma unroll
      for (int st = TM / 2; st > 0; st >>= 1)
#pragma unroll
        for (int i = 0; i < TM; ++i)
          if ((i & st) == 0) {
            const Word x = best[i], y = best[i + st];
            best[i] = max(x, y);
            best[i + st] = min(x, y);
          }
    }
  }
  // Entry `lane` (after meet), 0 past the list.
  __device__ Word mine() const {
    const int lane = threadIdx.x & 63;
    Word w = 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) w = i == lane ? best[i] : w;
    return w;
  }
  // Lane i takes entry i, and its place among the chosen ids; own >= 0 goes
  // behind them.
  __device__ void emit(int take, int32_t own, int slots, int32_t* out) const {
    const int lane = threadIdx.x & 63;
    const Word w = mine();
    const bool live = lane < take && w != 0;
    const uint32_t me = live ? static_cast<uint32_t>(id(w)) : 0xffffffffu;
    int n = __popcll(__ballot(live));
    int place = 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) place += static_cast<uint32_t>(__shfl(static_cast<int>(me), i)) < me ? 1 : 0;
    if (live) out[place] = static_cast<int32_t>(me);
    if (own >= 0 && lane == 0) out[n] = own;
    n += own >= 0;
    for (int i = n + lane; i < slots; i += 64) out[i] = -1;
  }
};

// How a type's scores are ranked.
template <typename T> struct Rank;
template <> struct Rank<bf16_t> { using Word = uint32_t; static constexpr bool kHalf = false; static constexpr int kWords = 1; };
template <> struct Rank<f16_t> { using Word = uint32_t; static constexpr bool kHalf = true; static constexpr int kWords = 1; };
template <> struct Rank<float> { using Word = uint64_t; static constexpr bool kHalf = false; static constexpr int kWords = 2; };

// The own block where it counts, else -1.
__device__ inline int32_t own_entry(const Paged& p, int current, int32_t seq, int32_t own) {
  return current && page_of(p, seq, own) >= 0 ? own : -1;
}

// The part-th run of a sequence's new tokens, at most `size` of them, inside
// the tokens [t0, t1). Parts are counted 64 sequences at a time by a wave's
// lanes.
struct Part {
  int32_t seq, begin, end;  // tokens; seq -1: no such part
};

__device__ inline Part find_part(const Paged& p, int32_t t0, int32_t t1, int32_t size, int32_t part) {
  const int lane = threadIdx.x & 63;
  int32_t before = 0, reach = 0;
  for (int32_t base = 0; base < p.seqs; base += 64) {
    const NewTokens r = counted_tokens(p, base, reach);
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
