// Which blocks new tokens attend to over a paged cache.
//
// score(j) = T(float32(q . kbar_j)) for the strictly past blocks j < own =
// position / block, the product exact; the `take` best by (score desc, block
// id asc), ids ascending, the own block last, -1 padding: the rules of
// gate.hip. A block without a page (a table entry outside the cache) never
// ranks, nor do scores of -inf and NaN.
//
// * score_kernel, select_kernel: every type and size, and few queries. All
//   scores in float64, over the whole chip, then one wave per query.
// * tiles_kernel: 16-bit types, many queries (below).
#include "paged_gate.h"
#include "paged_lds.h"

#include <type_traits>

#include "rotary.h"

namespace moba {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));

// Scores of one token's query heads of one kv head against a run of its past
// blocks: a block's representative belongs to D / 16 lanes, which hold it in
// float64 for the heads of the group. One token of each of 32 sequences of up to
// 100k keys, 32 and 8 heads of 128: 22 us, 3 rounds of workgroups, each a chain of
// lengths -> table -> representative and about as long again of conversions to
// float64 and products; its bytes take 5. (Sums over lanes one by one: the same.)
constexpr int kScoreThreads = 256;
constexpr int kScoreRows = 2;  // blocks per lane group, in flight together
template <typename T, int LPR>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(GateArgs a) {
  constexpr int D = 16 * LPR;
  constexpr int G = kScoreThreads / LPR;
  const int32_t local = blockIdx.x / a.h_kv;
  const int hk = blockIdx.x % a.h_kv;
  const TokenAt at = locate(a.p, a.tok0 + local);
  if (at.pos < 0) return;
  const int32_t own = at.pos / a.p.block;
  const int32_t past = own < a.p.width ? own : a.p.width;
  const int32_t j0 = blockIdx.y * (G * kScoreRows);
  if (j0 >= past) return;
  const int lane = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const RotLane rl = rot_lane(lane, 0, 0);
  const int group = a.h_q / a.h_kv;
  const int64_t row0 = static_cast<int64_t>(local) * a.h_q + hk * group;
  const T* q = static_cast<const T*>(a.q) + (static_cast<int64_t>(a.tok0) * a.h_q + row0) * D;
  int32_t page[kScoreRows];
#pragma unroll
  for (int i = 0; i < kScoreRows; ++i) {
    const int32_t j = j0 + i * G + g;
    page[i] = j < past ? page_of(a.p, at.seq, j) : -1;
  }
  double kd[kScoreRows][16];
#pragma unroll
  for (int i = 0; i < kScoreRows; ++i) {
    RawRow<T> raw;
    raw.load(static_cast<const T*>(a.kbar) + (static_cast<int64_t>(max(page[i], 0)) * a.h_kv + hk) * D, rl);
#pragma unroll
    for (int e = 0; e < 16; ++e) kd[i][e] = static_cast<double>(raw.element(e));
  }
  constexpr int H = 4;  // heads in flight
  for (int h0 = 0; h0 < group; h0 += H) {
    RawRow<T> raw[H];
#pragma unroll
    for (int u = 0; u < H; ++u) raw[u].load(q + min(h0 + u, group - 1) * D, rl);
    // Element i H + u is block i's and head u's share of this lane. The sums over
    // the lanes halve a lane's elements with every exchange, as long as it has
    // several: 7 exchanges at D = 128, not 24.
    constexpr int N = kScoreRows * H;
    double t[N] = {};
#pragma unroll
    for (int u = 0; u < H; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const double x = static_cast<double>(raw[u].element(e));
#pragma unroll
        for (int i = 0; i < kScoreRows; ++i) t[i * H + u] = fma(x, kd[i][e], t[i * H + u]);
      }
    int first = 0;  // the lane's elements are first, first + 1, ..
#pragma unroll
    for (int off = 1; off < LPR; off <<= 1) {
      const int left = N / (2 * off);
      if (left > 0) {
        const bool upper = lane & off;
        first += upper ? left : 0;
#pragma unroll
        for (int e = 0; e < left; ++e) {
          const double give = upper ? t[e] : t[e + left];
          t[e] = (upper ? t[e + left] : t[e]) + __shfl_xor(give, off);
        }
      } else {
        t[0] += __shfl_xor(t[0], off);
      }
    }
    if (lane < N) {
#pragma unroll
      for (int e = 0; e < (N / LPR > 0 ? N / LPR : 1); ++e) {
        const int i = (first + e) / H, u = (first + e) % H;
        const int32_t j = j0 + i * G + g;
        if (j < past && h0 + u < group) {
          int32_t pg = page[0];
#pragma unroll
          for (int x = 1; x < kScoreRows; ++x) pg = i == x ? page[x] : pg;
          a.keys[(row0 + h0 + u) * a.p.width + j] =
              pg < 0 ? 0u : score_key<Rank<T>>(Elem<T>::round(static_cast<float>(t[e])));
        }
      }
    }
  }
}

// The `take` best of a query's scores: one wave per (token, query head), each
// lane every 64th block.
template <typename T, int TM>
__global__ void __launch_bounds__(256) select_kernel(GateArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(a.slice) * a.h_q) return;
  const int lane = threadIdx.x & 63;
  const TokenAt at = locate(a.p, a.tok0 + static_cast<int32_t>(row / a.h_q));
  int32_t* out = a.block_idx + (static_cast<int64_t>(a.tok0) * a.h_q + row) * a.slots;
  if (at.pos < 0) {
    for (int i = lane; i < a.slots; i += 64) out[i] = -1;
    return;
  }
  const int32_t own = at.pos / a.p.block;
  const int32_t past = a.take ? (own < a.p.width ? own : a.p.width) : 0;
  WaveBest<Rank<T>, TM> list;
  list.clear();
  list.add_all(a.keys + row * a.p.width, past, lane, 64);
  list.meet();
  list.emit(a.take, own_entry(a.p, a.current, at.seq, own), a.slots, out);
}

// ---------------------------------------------------------------------------
// Many queries, 16-bit types. A wave holds 32 queries (tokens by the query
// heads of one kv head), two lanes each; the representatives pass through LDS
// 64 at a time, and two 32x32x16 MFMA chains leave each lane 2 x 16
// approximate scores of its query. |approximate - exact| <= E: the products
// are exact in float32, D additions round by at most a unit of the last place
// each (truncation included) of sums of at most |q| |kbar|. (The unit keeps
// subnormal inputs of both types, as it does subnormal float32 results: 16
// products of 2^-24 and 1 in fp16, of 2^-130 and 2^10 in bf16, of 2^-100 and
// 2^-40, come out exact.)
//
// Two passes over the blocks. The first keeps the largest of each lane's 16
// scores per tile, the best K of those: the take-th of both lanes' lists is a
// score that `take` blocks reach, so whatever cannot round to its key is out.
// The second writes the scores that can to a small buffer per lane (a few per
// query). A full buffer goes into the lane's list
// of the best M by (largest key the score can have, id), a key being the
// score rounded to the type, and the list's last entry then bounds what comes.
//
// An entry whose smallest key is its largest is certain, the others are
// marked. At the end a lane forms the exact scores of its marked entries, as
// far down as `take` certain ones do not stand above them, and the two lists
// are ranked. What left a list has no larger key than its last entry had, so
// the result stands where the last chosen entry ranks no lower than both
// lists' last; the other queries (constructed ties, infinities, NaN) score
// every block exactly.
//
// 2048 tokens of 32 and 8 heads of 128 over 1008 blocks, take 7, bf16: 90 us (the
// products of both passes take 28 at the rate of a large product; one pass that
// keeps sorted lists as it goes took 168 for the lists alone). What is left is
// VALU work at two waves per SIMD, which the grid has: the candidates and the
// exact scores. 3396 tokens of 12 sequences, 16 and 4 heads of 64 in fp16, take
// 11: 81 us.
constexpr int kNormParts = 16;

template <typename T> struct GateUnit;
template <> struct GateUnit<bf16_t> {
  typedef bf16x8_t vec;
  static constexpr float kLowest = -3.3961514e38f;  // rounds to -inf, as all below it
  static constexpr float kUnit = 0.008f;            // above the largest relative unit, 2^-7
  static constexpr float kSmall = 1e-37f;           // above the smallest absolute one
  __device__ static floatx16_t mma(vec a, vec b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // x rounded to the type, its bits in the upper half.
  __device__ static uint32_t bits(float x) {
    return f2u(static_cast<float>(static_cast<__bf16>(x)) + 0.f);
  }
  // The value of a rounded score's ordered bits.
  __device__ static float value(uint32_t upper) { return u2f(upper); }
};
template <> struct GateUnit<f16_t> {
  typedef f16x8_t vec;
  static constexpr float kLowest = -65520.f;
  static constexpr float kUnit = 0.001f;
  static constexpr float kSmall = 1e-7f;
  __device__ static floatx16_t mma(vec a, vec b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static uint32_t bits(float x) {
    const _Float16 r = static_cast<_Float16>(x) + static_cast<_Float16>(0);
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, r)) << 16;
  }
  __device__ static float value(uint32_t upper) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(upper >> 16)));
  }
};

// Order of 16-bit floats in the upper half of a word, and back.
__device__ inline uint32_t ordered(uint32_t u) {
  return (u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u)) & 0xffff0000u;
}
__device__ inline uint32_t unordered(uint32_t o) {
  return (o & 0x80000000u ? o ^ 0x80000000u : ~o) & 0xffff0000u;
}

__device__ inline uint32_t med3(uint32_t a, uint32_t b, uint32_t c) {
  return max(min(a, b), min(max(a, b), c));
}

// The largest |kbar| of every (sequence, kv head)'s past blocks, in kNormParts
// parts, as float bits (NaN largest). grid (seqs * h_kv, kNormParts).
template <typename T, int LPR>
__global__ void __launch_bounds__(256) norm_kernel(GateArgs a) {
  constexpr int D = 16 * LPR;
  __shared__ uint32_t s_best[4];
  const int32_t seq = blockIdx.x / a.h_kv;
  const int hk = blockIdx.x % a.h_kv;
  const NewTokens r = new_tokens(a.p, seq);
  const int32_t past = r.n ? min((r.len - 1) / a.p.block, a.p.width) : 0;
  const RotLane rl = rot_lane(threadIdx.x % LPR, 0, 0);
  uint32_t best = 0;
  for (int32_t j = blockIdx.y * (256 / LPR) + threadIdx.x / LPR; j < past; j += kNormParts * (256 / LPR)) {
    const int32_t page = page_of(a.p, seq, j);
    if (page < 0) continue;
    RawRow<T> raw;
    raw.load(static_cast<const T*>(a.kbar) + (static_cast<int64_t>(page) * a.h_kv + hk) * D, rl);
    float v[16];
    raw.widen(v);
    best = max(best, f2u(sqrtf(row_sum<LPR>(square_sum(v)))) & 0x7fffffffu);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) best = max(best, static_cast<uint32_t>(__shfl_xor(static_cast<int>(best), off)));
  if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0)
    a.norms[static_cast<int64_t>(blockIdx.x) * kNormParts + blockIdx.y] =
        max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
}

// Exact key of one block, by one lane.
template <typename T, int D>
__device__ inline uint32_t exact_key(const T* q, const T* kb) {
  double t = 0.0;
  for (int d = 0; d < D; d += 8) {
    const u32x4 qa = *reinterpret_cast<const u32x4*>(q + d);
    const u32x4 ka = *reinterpret_cast<const u32x4*>(kb + d);
    const T* qe = reinterpret_cast<const T*>(&qa);
    const T* ke = reinterpret_cast<const T*>(&ka);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      t = fma(static_cast<double>(Elem<T>::load(qe, e)), static_cast<double>(Elem<T>::load(ke, e)), t);
  }
  return score_key<Rank<T>>(Elem<T>::round(static_cast<float>(t)));
}

// A query's blocks all scored exactly, by one wave. Arguments by value: a
// reference would put the caller's copy into scratch memory.
template <typename T, int D, int TM>
__device__ __attribute__((noinline)) void exact_query(const int32_t* pages, int32_t n_pages, int32_t past,
                                                      const T* kbar, int64_t page_stride, const T* q,
                                                      int take, int32_t own, int slots, int32_t* out) {
  WaveBest<Rank<T>, TM> list;
  list.clear();
  for (int32_t j = threadIdx.x & 63; j < past; j += 64) {
    const int32_t page = pages[j];
    if (page >= 0 && page < n_pages) list.add(list.word(exact_key<T, D>(q, kbar + page * page_stride), j));
  }
  list.meet();
  list.emit(take, own, slots, out);
}

// What a wave's lanes wrote to LDS, visible to its other lanes.
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kBuffer = 24;  // entries per lane

template <typename T, int D, int M, int K>
__global__ void __launch_bounds__(256, 2) tiles_kernel(GateArgs a) {
  using U = GateUnit<T>;
  using V8 = typename U::vec;
  constexpr int RQ = D / 8;     // 16-byte pieces per row
  constexpr int ROWS = 64;      // representatives per stage
  constexpr int KS = D / 16;
  // Aligned to the rows, whose bits the exclusive ors of the reads change.
  __shared__ __attribute__((aligned(512))) uint16_t rows[2][ROWS * D];
  __shared__ int32_t s_page[2][ROWS];
  __shared__ int32_t s_valid[4][2];
  constexpr int kHeld = M > kBuffer ? M : kBuffer;
  __shared__ float s_score[4][kHeld][64];
  __shared__ uint16_t s_id[4][kHeld][64];
  const Part pt = find_part(a.p, 0, a.p.tokens, a.tile_tokens, blockIdx.x);
  if (pt.seq < 0) return;
  const NewTokens nt = new_tokens(a.p, pt.seq);
  const int hk = blockIdx.y, group = a.h_q / a.h_kv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int n_rows = (pt.end - pt.begin) * group;
  const int mine = wave * 32 + (lane & 31);
  const bool live = mine < n_rows;
  const bool busy = wave * 32 < n_rows;  // the wave has queries
  const int32_t tok = pt.begin + (live ? mine : 0) / group;
  const int64_t qrow = static_cast<int64_t>(tok) * a.h_q + hk * group + (live ? mine : 0) % group;
  const T* q = static_cast<const T*>(a.q) + qrow * D;
  const int32_t pos0 = nt.len - nt.n - nt.first;  // a token's position: pos0 + token
  const int32_t own = (pos0 + tok) / a.p.block;
  const int32_t past = live ? min(own, a.p.width) : 0;
  const int32_t horizon = min((pos0 + pt.end - 1) / a.p.block, a.p.width);
  const int32_t sure = min((pos0 + pt.begin) / a.p.block, a.p.width);  // past for every query here
  const int stages = (horizon + ROWS - 1) / ROWS;

  V8 bq[KS];
  float qn = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    bq[k] = __builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(q + 16 * k + 8 * h));
#pragma unroll
    for (int e = 0; e < 8; ++e) qn = fmaf(static_cast<float>(bq[k][e]), static_cast<float>(bq[k][e]), qn);
  }
  // Norms carry 2e-18 on top: up to 256 squares of less than 2^-126 each
  // may be missing from their sums.
  qn = sqrtf(qn + __shfl_xor(qn, 32)) * 1.0001f + 2e-18f;
  float kn = 0.f;
  {
    uint32_t best = 0;
    const uint32_t* norms = a.norms + (static_cast<int64_t>(pt.seq) * a.h_kv + hk) * kNormParts;
#pragma unroll
    for (int i = 0; i < kNormParts; ++i) best = max(best, norms[i]);
    kn = u2f(best) * 1.0001f + 2e-18f;
  }
  // Widened by the rounding of a -+ E itself, with |a| * 2.4e-7 below.
  const float E = (qn * kn * (D * 0x1p-23f) + (D + 1) * 1.2e-38f) * 1.001f;
  const bool bounded = qn * kn < 3e38f && E < 3e38f;  // false for infinities and NaN

  // Pages of stage st, by wave 0: to LDS, with a bit for each that is one.
  const int32_t* pages = a.p.table + static_cast<int64_t>(pt.seq) * a.p.width;
  auto page_at = [&](int st) { return pages[min(st * ROWS + lane, horizon - 1)]; };
  auto put_pages = [&](int st, int32_t page) {
    const bool is = st * ROWS + lane < horizon && page >= 0 && page < a.p.pages;
    const uint64_t ok = __ballot(is);
    s_page[st & 1][lane] = is ? page : 0;
    if (lane == 0) {
      s_valid[st & 3][0] = static_cast<int32_t>(ok);
      s_valid[st & 3][1] = static_cast<int32_t>(ok >> 32);
    }
  };
  auto stage = [&](int st) {
    int32_t page[ROWS * RQ / 256];
#pragma unroll
    for (int u = 0; u < ROWS * RQ / 256; ++u) page[u] = s_page[st & 1][(u * 256 + tid) / RQ];
#pragma unroll
    for (int u = 0; u < ROWS * RQ / 256; ++u) {
      const int i = u * 256 + tid, row = i / RQ, piece = i % RQ;
      const T* src = static_cast<const T*>(a.kbar) + (static_cast<int64_t>(page[u]) * a.h_kv + hk) * D +
                     8 * (piece ^ swizzle_rows<D>(row));
      load_to_lds(src, &rows[st & 1][(u * 256 + wave * 64) * 8]);
    }
  };

  // Representatives lane & 31 and 32 more: feature step 0 of the first stage.
  const uint32_t k_at0 = lds_address(&rows[0][(lane & 31) * D + 8 * (h ^ swizzle_rows<D>(lane & 31))]);
  uint32_t key[M];
#pragma unroll
  for (int i = 0; i < M; ++i) key[i] = 0;
  float tops[K];  // pass 0: the best tile maxima, best first
#pragma unroll
  for (int i = 0; i < K; ++i) tops[i] = -INFINITY;
  float floor_value = U::kLowest;  // pass 1: scores that round to at most this are out
  int held = 0;                    // entries in the lane's buffer
  float* score = &s_score[wave][0][lane];  // entry i at [64 i]
  uint16_t* id = &s_id[wave][0][lane];
  // The buffer into the list.
  auto fold = [&]() {
    for (int i = 0; __any(i < held); ++i) {
      const float x = score[64 * i];
      const uint32_t top = U::bits(fmaf(fabsf(x), 2.4e-7f, x) + E);
      const uint32_t low = U::bits(fmaf(-fabsf(x), 2.4e-7f, x) - E);
      uint32_t e = ordered(top) | (0x7fffu - id[64 * i]) << 1 | (top != low ? 1u : 0u);
      e = i < held ? e : 0u;
#pragma unroll
      for (int p = M - 1; p > 0; --p) key[p] = med3(key[p - 1], key[p], e);
      key[0] = max(key[0], e);
    }
    held = 0;
    if (key[M - 1]) floor_value = fmaxf(floor_value, U::value(unordered(key[M - 1])));
  };
  for (int pass = 0; pass < 2 && stages > 0; ++pass) {
    __syncthreads();  // the previous pass is done with the stages
    if (wave == 0) {
      put_pages(0, page_at(0));
      if (stages > 1) put_pages(1, page_at(1));
    }
    __syncthreads();
    stage(0);
    for (int st = 0; st < stages; ++st) {
      wait_loads<0>();
      meet();
      int32_t ahead = -1;
      if (wave == 0 && st + 2 < stages) ahead = page_at(st + 2);
      if (st + 1 < stages) stage(st + 1);
      if (busy) {
        const uint32_t valid[2] = {static_cast<uint32_t>(read_word(&s_valid[st & 3][0])),
                                   static_cast<uint32_t>(read_word(&s_valid[st & 3][1]))};
        floatx16_t s[2] = {floatx16_t{}, floatx16_t{}};
        const uint32_t k_at = k_at0 + (st & 1) * ROWS * D * 2;
        auto step = [&](auto kc) {
          constexpr int k = decltype(kc)::value;
          u32x4 x[4];
          read_row_pairs<64 * k, 32 * D * 2>(k_at, x);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            s[u & 1] = U::mma(__builtin_bit_cast(V8, x[u]), bq[2 * k + (u >> 1)], s[u & 1]);
        };
        steps(std::make_integer_sequence<int, KS / 2>{}, step);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int32_t j0 = st * ROWS + half * 32;
          if (j0 >= horizon) continue;
          const uint32_t ok = valid[half];
          if (j0 + 32 > sure || ok != 0xffffffffu) {  // some blocks are not for every query
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const int o = 8 * (v >> 2) + 4 * h + (v & 3);
              if (j0 + o >= past || !((ok >> o) & 1u)) s[half][v] = -INFINITY;
            }
          }
          float most = s[half][0];
#pragma unroll
          for (int v = 1; v < 16; ++v) most = fmaxf(most, s[half][v]);
          if (pass == 0) {
#pragma unroll
            for (int i = K - 1; i > 0; --i) tops[i] = __builtin_amdgcn_fmed3f(tops[i - 1], tops[i], most);
            tops[0] = fmaxf(tops[0], most);
          } else if (__any(fmaf(fabsf(most), 2.4e-7f, most) + E > floor_value)) {
            if (__any(held > kBuffer - 16)) fold();
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              // Written whether it counts or not: about half of these tests
              // hold for some lane.
              const float x = s[half][v];
              score[64 * held] = x;
              id[64 * held] = static_cast<uint16_t>(j0 + 8 * (v >> 2) + 4 * h + (v & 3));
              held += fmaf(fabsf(x), 2.4e-7f, x) + E > floor_value ? 1 : 0;
            }
          }
        }
      }
      if (wave == 0 && st + 2 < stages) put_pages(st + 2, ahead);
    }
    if (pass == 0 && busy) {
      // The take-th of both lists: the best over i of the lower of one's i-th
      // and the other's (take - i)-th.
      float other[K], bound = -INFINITY;
#pragma unroll
      for (int i = 0; i < K; ++i) other[i] = __shfl_xor(tops[i], 32);
#pragma unroll
      for (int i = 0; i <= K; ++i) {
        float theirs = INFINITY;
#pragma unroll
        for (int u = 0; u < K; ++u) theirs = u == a.take - i - 1 ? other[u] : theirs;
        if (i <= a.take) bound = fmaxf(bound, fminf(i ? tops[i - 1] : INFINITY, theirs));
      }
      // A key is within a unit of its score, so what can reach the bound's
      // lowest key lies above one unit (2^-7 of it in bf16, 2^-10 in fp16)
      // below the bound's lowest value.
      const float low = fmaf(-fabsf(bound), 2.4e-7f, bound) - E;
      const float edge = low - fabsf(low) * U::kUnit - U::kSmall;
      if (edge > floor_value) floor_value = edge;
    }
  }
  if (!busy) return;
  fold();

  const uint32_t last = key[M - 1];
  bool settled = bounded || past == 0;
  // Exact scores of marked entries that `take` certain ones do not outrank:
  // listed over the wave, then D / 16 lanes to each.
  {
    uint32_t* value = reinterpret_cast<uint32_t*>(&s_score[wave][0][0]);  // [entry][lane]
    uint16_t* list = &s_id[wave][0][0];                                   // lane | entry << 6
    uint64_t wanted = 0;
    int certain = 0, n_list = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const bool marked = key[i] & 1u;
      // Only the wave's queries: the other lanes hold leavings of its first row.
      const bool want = marked && live && settled && certain < a.take;
      certain += key[i] && !marked;
      const uint64_t mask = __ballot(want);
      if (want) {
        list[n_list + __popcll(mask & ((uint64_t(1) << lane) - 1))] = static_cast<uint16_t>(lane | i << 6);
        value[64 * i + lane] = key[i];
        wanted |= uint64_t(1) << i;
      }
      n_list += __popcll(mask);
      key[i] &= ~1u;
    }
    wave_sync();
    constexpr int LPR = D / 16;
    const RotLane rl = rot_lane(lane % LPR, 0, 0);
    for (int p0 = 0; p0 < n_list; p0 += 64 / LPR) {
      const int p = p0 + lane / LPR;
      const int code = list[min(p, n_list - 1)];
      const int l = code & 63, at = 64 * (code >> 6) + l;
      const uint32_t entry = value[at];
      const int row = wave * 32 + (l & 31);
      const int64_t qr = static_cast<int64_t>(pt.begin + row / group) * a.h_q + hk * group + row % group;
      const int32_t page = max(page_of(a.p, pt.seq, static_cast<int32_t>(0x7fffu - ((entry >> 1) & 0x7fffu))), 0);
      RawRow<T> rq, rk;
      rq.load(static_cast<const T*>(a.q) + qr * D, rl);
      rk.load(static_cast<const T*>(a.kbar) + (static_cast<int64_t>(page) * a.h_kv + hk) * D, rl);
      double t = 0.0;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        t = fma(static_cast<double>(rq.element(e)), static_cast<double>(rk.element(e)), t);
#pragma unroll
      for (int off = 1; off < LPR; off <<= 1) t += __shfl_xor(t, off);
      const uint32_t x = score_key<Rank<T>>(Elem<T>::round(static_cast<float>(t)));
      if (lane % LPR == 0 && p < n_list) value[at] = x ? x | (entry & 0xfffeu) : 0u;
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < M; ++i)
      if ((wanted >> i) & 1) key[i] = value[64 * i + lane];
  }
  // Ranks among both lanes' entries.
  uint32_t other[M];
#pragma unroll
  for (int i = 0; i < M; ++i) other[i] = static_cast<uint32_t>(__shfl_xor(static_cast<int>(key[i]), 32));
  uint32_t lowest = 0xffffffffu;  // the lowest chosen entry
  int n = 0;
  uint64_t chosen = 0;            // bits of this lane's chosen entries
#pragma unroll
  for (int i = 0; i < M; ++i) {
    int rank = 0;
#pragma unroll
    for (int u = 0; u < M; ++u) rank += (key[u] > key[i]) + (other[u] > key[i]);
    if (key[i] && rank < a.take) {
      chosen |= uint64_t(1) << i;
      lowest = min(lowest, key[i]);
      ++n;
    }
  }
  n += __shfl_xor(n, 32);
  lowest = min(lowest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(lowest), 32)));
  const uint32_t out_of = max(last, static_cast<uint32_t>(__shfl_xor(static_cast<int>(last), 32)));
  if (out_of && (n < a.take || lowest < (out_of & ~1u))) settled = false;

  // Places in the order of the ids: larger (0x7fff - id) first, 0 for entries
  // that are not chosen (ids are below 0x7fff).
  int32_t* out = a.block_idx + qrow * a.slots;
  const uint64_t theirs = __shfl_xor(static_cast<unsigned long long>(chosen), 32);
#pragma unroll
  for (int i = 0; i < M; ++i) {
    key[i] = (chosen >> i) & 1u ? key[i] & 0xfffeu : 0u;
    other[i] = (theirs >> i) & 1u ? other[i] & 0xfffeu : 0u;
  }
  if (settled && live) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (!key[i]) continue;
      int place = 0;
#pragma unroll
      for (int u = 0; u < M; ++u) place += (key[u] > key[i]) + (other[u] > key[i]);
      out[place] = static_cast<int32_t>(0x7fffu - (key[i] >> 1));
    }
    if (h == 0) {
      const int32_t o = own_entry(a.p, a.current, pt.seq, own);
      if (o >= 0) out[n++] = o;
      for (; n < a.slots; ++n) out[n] = -1;
    }
  }
  uint64_t open = __ballot(!settled && live && h == 0);
  while (open) {
    const int l = __builtin_ctzll(open);
    open &= open - 1;
    const int row = wave * 32 + l;
    const int32_t t = pt.begin + row / group;
    const int64_t qr = static_cast<int64_t>(t) * a.h_q + hk * group + row % group;
    const int32_t o = (pos0 + t) / a.p.block;
    exact_query<T, D, K>(a.p.table + static_cast<int64_t>(pt.seq) * a.p.width, a.p.pages, min(o, a.p.width),
                         static_cast<const T*>(a.kbar) + hk * D, static_cast<int64_t>(a.h_kv) * D,
                         static_cast<const T*>(a.q) + qr * D, a.take,
                         own_entry(a.p, a.current, pt.seq, o), a.slots, a.block_idx + qr * a.slots);
  }
}

// Rows of no sequence: all -1. One wave per token.
__global__ void __launch_bounds__(64) nobody_kernel(GateArgs a) {
  const int32_t tok = a.tok0 + static_cast<int32_t>(blockIdx.x);
  if (locate(a.p, tok).pos >= 0) return;
  int32_t* out = a.block_idx + static_cast<int64_t>(tok) * a.h_q * a.slots;
  for (int i = threadIdx.x; i < a.h_q * a.slots; i += 64) out[i] = -1;
}

// The tiles from kTileRows query rows on, where sequences have several tokens (a
// tile holds one sequence's). bf16, 32 and 8 heads of 128, tiles and score +
// select: 32 sequences of 256 blocks, 4 new tokens each (4096 rows) 36 and 32
// us, 8 each 37 and 58; 4 of 512 blocks, 32 tokens each (4096 rows) 47 and 58;
// one of 512 blocks, 64 tokens (2048 rows) 46 and 32. 8 heads of 64, 8
// sequences of 64 blocks, 64 tokens each (4096 rows) 21 and 31, 8 each 21 and 16.
constexpr int64_t kTileRows = 4096;
constexpr int64_t kMaxBlocks = int64_t(1) << 24;  // workgroups of 256 threads: a launch holds fewer than 2^32
bool tiles_take(const moba_paged& c) {
  return c.dtype != MOBA_FP32 && c.take > 0 && c.table_width < (1 << 15) && c.h_q / c.h_kv <= 128 &&
         c.h_kv <= 65535 && c.tokens >= 4 * c.seqs && c.tokens * c.h_q >= kTileRows &&
         c.seqs * c.h_kv < kMaxBlocks && c.tokens / (128 / (c.h_q / c.h_kv)) + c.seqs < kMaxBlocks;
}

int64_t score_slice(const moba_paged& c) {
  int64_t n = (int64_t(1) << 24) / (c.h_q * c.table_width);
  if (n * c.h_kv >= kMaxBlocks) n = kMaxBlocks / 2 / c.h_kv;
  return n < 1 ? 1 : (n < c.tokens ? n : c.tokens);
}

template <typename F>
int with_dim(const moba_paged& c, F&& go) {
  return MOBA_DISPATCH_DTYPE(static_cast<int>(c.dtype), T, [&] {
    switch (c.head_dim) {
      case 64: return go(T{}, std::integral_constant<int, 64>{});
      case 128: return go(T{}, std::integral_constant<int, 128>{});
      default: return go(T{}, std::integral_constant<int, 256>{});
    }
  });
}

int run_tiles(const moba_paged& c, GateArgs a, bool all_rows, hipStream_t s) {
  const int64_t group = c.h_q / c.h_kv;
  a.tile_tokens = static_cast<int>(128 / group);
  const int64_t parts = cdiv(c.tokens, a.tile_tokens) + c.seqs;
  return with_dim(c, [&](auto t, auto dim) {
    using T = decltype(t);
    constexpr int D = decltype(dim)::value;
    if constexpr (sizeof(T) == 2) {
      hipLaunchKernelGGL((norm_kernel<T, D / 16>), dim3(static_cast<unsigned>(c.seqs * c.h_kv), kNormParts),
                         dim3(256), 0, s, a);
      for (int64_t t0 = 0; all_rows && t0 < c.tokens; t0 += kMaxBlocks) {
        a.tok0 = static_cast<int32_t>(t0);
        const int64_t n = c.tokens - t0 < kMaxBlocks ? c.tokens - t0 : kMaxBlocks;
        hipLaunchKernelGGL(nobody_kernel, dim3(static_cast<unsigned>(n)), dim3(64), 0, s, a);
      }
      auto go = [&](auto m, auto tm) {
        hipLaunchKernelGGL((tiles_kernel<T, D, decltype(m)::value, decltype(tm)::value>),
                           dim3(static_cast<unsigned>(parts), static_cast<unsigned>(c.h_kv)), dim3(256), 0, s, a);
        return check_launch("moba_paged_gate (tiles)");
      };
      using std::integral_constant;
      if (c.take <= 8) return go(integral_constant<int, 12>{}, integral_constant<int, 8>{});
      if (c.take <= 16) return go(integral_constant<int, 20>{}, integral_constant<int, 16>{});
      return go(integral_constant<int, 36>{}, integral_constant<int, 32>{});
    } else {
      return fail(MOBA_ERR_UNSUPPORTED, "unreachable");
    }
  });
}

}  // namespace

// Up to 1024 query rows the attention chooses from the scores itself: 1024 of
// bf16 over 390 blocks on average 117 us, with select_kernel 121; 4000 of float32
// over 130 blocks 89 and 74.
bool scores_only(const moba_paged& c) {
  return !tiles_take(c) && c.tokens * c.h_q <= 1024 && score_slice(c) == c.tokens;
}

size_t gate_workspace(const moba_paged& c) {
  const size_t n = tiles_take(c) ? static_cast<size_t>(c.seqs * c.h_kv * kNormParts)
                                 : static_cast<size_t>(score_slice(c) * c.h_q * c.table_width);
  return (4 * n + 255) & ~size_t(255);
}

static GateArgs gate_args(const moba_paged& c, const Paged& p, void* workspace) {
  GateArgs a;
  a.p = p;
  a.q = c.q;
  a.kbar = c.kbar;
  a.keys = a.norms = static_cast<uint32_t*>(workspace);
  a.block_idx = c.block_idx;
  a.h_q = static_cast<int>(c.h_q);
  a.h_kv = static_cast<int>(c.h_kv);
  a.slots = static_cast<int>(c.slots);
  a.take = static_cast<int>(c.take);
  a.current = c.always_current != 0;
  return a;
}

// Scores of tokens [a.tok0, a.tok0 + a.slice).
static int run_scores(const moba_paged& c, const GateArgs& a, hipStream_t s) {
  if (c.take == 0) return MOBA_OK;
  return with_dim(c, [&](auto t, auto dim) {
    constexpr int LPR = decltype(dim)::value / 16;
    const int64_t tiles = cdiv(c.table_width, kScoreThreads / LPR * kScoreRows);
    if (tiles > 65535) return fail(MOBA_ERR_UNSUPPORTED, "block table too wide");
    hipLaunchKernelGGL((score_kernel<decltype(t), LPR>),
                       dim3(static_cast<unsigned>(a.slice * c.h_kv), static_cast<unsigned>(tiles)),
                       dim3(kScoreThreads), 0, s, a);
    return check_launch("moba_paged_gate (scores)");
  });
}

int gate_scores(const moba_paged& c, const Paged& p, void* workspace, hipStream_t s) {
  GateArgs a = gate_args(c, p, workspace);
  a.tok0 = 0;
  a.slice = static_cast<int32_t>(c.tokens);
  return run_scores(c, a, s);
}

int gate_run(const moba_paged& c, const Paged& p, void* workspace, bool all_rows, hipStream_t s) {
  GateArgs a = gate_args(c, p, workspace);
  if (tiles_take(c)) return run_tiles(c, a, all_rows, s);
  const int64_t slice = score_slice(c);
  for (int64_t t0 = 0; t0 < c.tokens; t0 += slice) {
    a.tok0 = static_cast<int32_t>(t0);
    a.slice = static_cast<int32_t>(c.tokens - t0 < slice ? c.tokens - t0 : slice);
    int st = run_scores(c, a, s);
    if (st) return st;
    st = MOBA_DISPATCH_DTYPE(static_cast<int>(c.dtype), T, [&] {
      const dim3 grid(static_cast<unsigned>(cdiv(a.slice * c.h_q, 4)));
      if (c.take <= 8) hipLaunchKernelGGL((select_kernel<T, 8>), grid, dim3(256), 0, s, a);
      else if (c.take <= 16) hipLaunchKernelGGL((select_kernel<T, 16>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((select_kernel<T, 32>), grid, dim3(256), 0, s, a);
      return check_launch("moba_paged_gate (select)");
    });
    if (st) return st;
  }
  return MOBA_OK;
}

}  // namespace moba
