// Attention of chunks of new tokens over a paged cache, 16-bit types.
//
// Many queries choose the same block, so the work goes block by block: the
// (query, slot) entries of block_idx are sorted into columns, one per
// (sequence, kv head, block), a block's keys and values are staged in LDS once
// for up to kItem of its entries, and each entry leaves an un-normalised
// partial row that a last pass merges per query.
//
//   count   entries per (part of the tokens, kv head, block)
//   scan    first place of every (part, block), and the list of work items
//   place   entries to their places
//   attend  one work item (a block and up to kItem entries) at a time
//   merge   the slots of every query
//
// 2048 tokens at the end of 129k, 32 and 8 heads of 128 in bf16, 8 blocks of 128
// per query (0.5 million entries, 0.5 GB of keys and values that are each staged
// once): 9 + 14 + 10 us of sorting, 208 of attention, 56 of merging. The
// attention moves 0.8 GB, 3.8 TB/s: columns hold 64 entries on average, so half
// of a workgroup's waves wait for the next block, and two workgroups share a CU's
// LDS. The merge reads 0.27 GB of partial rows, 5.2 TB/s. 12 sequences with 1 to
// 700 tokens, 16 and 4 heads of 64 in fp16, 12 blocks of 64: 24, 104 and 32 us.
//
// An entry is its index in block_idx, which is also the index of its partial
// row. Entries of a column stand in no particular order; nothing depends on it.
#include "paged_chunk.h"

#include <utility>

#include "paged_gate.h"
#include "paged_lds.h"

namespace moba {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));

template <typename T> struct Unit;
template <> struct Unit<bf16_t> {
  typedef bf16x8_t vec;
  typedef __bf16 scalar;
  static constexpr uint32_t kInf = 0x7f80u;
  static constexpr float kShift = 0.f;
  __device__ static floatx16_t mma(vec a, vec b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Unit<f16_t> {
  typedef f16x8_t vec;
  typedef _Float16 scalar;
  static constexpr uint32_t kInf = 0x7c00u;
  static constexpr float kShift = 15.f;  // weights up to 2^15: the second parts of small ones stay in range
  __device__ static floatx16_t mma(vec a, vec b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Entries of a work item: one group of 32 for each of the four waves.
constexpr int kItem = 128;

// The block an entry of sequence `seq` attends to, or -1: padding, a block
// without a page or behind the sequence's last token.
__device__ inline int32_t entry_block(const Paged& p, int32_t seq, int32_t blk) {
  if (blk < 0 || static_cast<int64_t>(blk) * p.block >= p.seq_lens[seq]) return -1;
  return page_of(p, seq, blk) < 0 ? -1 : blk;
}

// Entries i0 + kSortThreads u of a part and kv head, kFlight of them in flight: their
// index in the slice and their block (-1: none, or past the last of n).
constexpr int kSortThreads = 1024;
constexpr int kFlight = 8;
__device__ inline void load_entries(const ChunkArgs& a, const Part& pt, int hk, int i0, int n,
                                    int32_t (&e)[kFlight], int32_t (&blk)[kFlight]) {
  const uint32_t group = a.h_q / a.h_kv, per = group * a.slots;
  const int32_t* ids = a.block_idx + static_cast<int64_t>(a.t0) * a.h_q * a.slots;
#pragma unroll
  for (int u = 0; u < kFlight; ++u) {
    const uint32_t i = min(i0 + kSortThreads * u, n - 1), t = i / per;
    e[u] = ((pt.begin - a.t0 + t) * a.h_q + hk * group) * a.slots + (i - t * per);
    blk[u] = ids[e[u]];
  }
#pragma unroll
  for (int u = 0; u < kFlight; ++u) blk[u] = i0 + kSortThreads * u < n ? entry_block(a.p, pt.seq, blk[u]) : -1;
}

// counts[part, kv head, block]; dynamic LDS: width counters. grid (parts, h_kv).
__global__ void __launch_bounds__(kSortThreads) column_count_kernel(ChunkArgs a) {
  extern __shared__ int32_t bins[];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.n_items = 0;
  const Part pt = find_part(a.p, a.t0, a.t1, a.part, blockIdx.x);
  if (pt.seq < 0) return;
  const int hk = blockIdx.y, group = a.h_q / a.h_kv, per = group * a.slots;
  for (int j = threadIdx.x; j < a.p.width; j += kSortThreads) bins[j] = 0;
  __syncthreads();
  const int n = (pt.end - pt.begin) * per;
  for (int i0 = threadIdx.x; i0 < n; i0 += kSortThreads * kFlight) {
    int32_t e[kFlight], blk[kFlight];
    load_entries(a, pt, hk, i0, n, e, blk);
#pragma unroll
    for (int u = 0; u < kFlight; ++u)
      if (blk[u] >= 0) atomicAdd(&bins[blk[u]], 1);
  }
  __syncthreads();
  int32_t* out = a.table + (static_cast<int64_t>(blockIdx.x) * a.h_kv + hk) * a.p.width;
  for (int j = threadIdx.x; j < a.p.width; j += kSortThreads) out[j] = bins[j];
}

// Per (sequence, kv head): table -> the place of every (part, block)'s first
// entry; work items of the columns. Dynamic LDS: width counters. grid (seqs,
// h_kv).
__global__ void __launch_bounds__(1024) column_scan_kernel(ChunkArgs a) {
  extern __shared__ int32_t sizes[];
  __shared__ int32_t wsum[2][16];
  __shared__ int32_t base_item;
  const int32_t seq = blockIdx.x;
  const int hk = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // This sequence's parts and where its entries begin.
  int32_t first = 0, lo = 0, hi = 0, len = 0, reach = 0;
  for (int32_t base = 0; base <= seq; base += 64) {
    const NewTokens o = counted_tokens(a.p, base, reach);
    const int32_t l = max(o.first, a.t0), h = min(o.first + o.n, a.t1);
    int32_t mine = base + lane < seq && h > l ? (h - l + a.part - 1) / a.part : 0;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mine += __shfl_xor(mine, off);
    first += mine;
    const int at = seq - base;  // below 64 in the last round
    lo = __shfl(l, at & 63);
    hi = __shfl(h, at & 63);
    len = __shfl(o.len, at & 63);
  }
  if (hi <= lo) return;
  const int32_t parts = (hi - lo + a.part - 1) / a.part;
  const int per = a.h_q / a.h_kv * a.slots;
  const int32_t place0 = (lo - a.t0) * a.h_q * a.slots + hk * (hi - lo) * per;
  const uint32_t row = a.h_kv * a.p.width;  // the table has at most 2^22 entries, or one part per sequence
  int32_t* table = a.table + static_cast<int64_t>(first) * row + static_cast<int64_t>(hk) * a.p.width;
  const int32_t blocks = min(a.p.width, (len - 1) / a.p.block + 1);  // lengths up to 2^31 - 1
  // The columns' entries into LDS, and the number of items; then the lists.
  int32_t items = 0;
  for (int round = 0; round < 2; ++round) {
    int32_t carry_e = 0, carry_i = 0;
    for (int32_t b0 = 0; b0 < blocks; b0 += 1024) {
      const int32_t b = b0 + threadIdx.x;
      int32_t n = 0;
      if (b < blocks) {
        if (round == 0) {
          const int32_t* p = table + b;
          for (int32_t q0 = 0; q0 < parts; q0 += 8) {
            int32_t x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = p[static_cast<int64_t>(min(q0 + u, parts - 1)) * row];
#pragma unroll
            for (int u = 0; u < 8; ++u) n += q0 + u < parts ? x[u] : 0;
          }
          sizes[b] = n;
        } else {
          n = sizes[b];
        }
      }
      const int32_t k = (n + kItem - 1) / kItem;
      int32_t ie = n, ii = k;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int32_t ye = __shfl_up(ie, off), yi = __shfl_up(ii, off);
        if (lane >= off) { ie += ye; ii += yi; }
      }
      if (lane == 63) { wsum[0][wave] = ie; wsum[1][wave] = ii; }
      __syncthreads();
      int32_t te = 0, ti = 0;
      for (int w = 0; w < 16; ++w) {
        if (w < wave) { ie += wsum[0][w]; ii += wsum[1][w]; }
        te += wsum[0][w];
        ti += wsum[1][w];
      }
      __syncthreads();
      if (round == 1 && b < blocks && n) {
        int32_t at = place0 + carry_e + ie - n;
        const int32_t i0 = base_item + carry_i + ii - k;
        for (int32_t i = 0; i < k && i0 + i < a.max_items; ++i)
          a.items[i0 + i] = make_int4(seq * a.h_kv + hk, b, at + i * kItem, min(kItem, n - i * kItem));
        int32_t* p = table + b;
        for (int32_t q0 = 0; q0 < parts; q0 += 8) {
          int32_t x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = p[static_cast<int64_t>(min(q0 + u, parts - 1)) * row];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (q0 + u < parts) {
              p[static_cast<int64_t>(q0 + u) * row] = at;
              at += x[u];
            }
          }
        }
      }
      carry_e += te;
      carry_i += ti;
    }
    items = carry_i;
    if (round == 0) {
      if (threadIdx.x == 0) base_item = atomicAdd(a.n_items, items);
      __syncthreads();
    }
  }
}

// Entries to their places; those that attend to nothing leave (m, l) = (-inf,
// 0). Dynamic LDS: width cursors. grid (parts, h_kv).
__global__ void __launch_bounds__(kSortThreads) column_place_kernel(ChunkArgs a) {
  extern __shared__ int32_t cursor[];
  const Part pt = find_part(a.p, a.t0, a.t1, a.part, blockIdx.x);
  if (pt.seq < 0) return;
  const int hk = blockIdx.y, group = a.h_q / a.h_kv, per = group * a.slots;
  const int32_t* row = a.table + (static_cast<int64_t>(blockIdx.x) * a.h_kv + hk) * a.p.width;
  for (int j = threadIdx.x; j < a.p.width; j += kSortThreads) cursor[j] = row[j];
  __syncthreads();
  const int n = (pt.end - pt.begin) * per;
  for (int i0 = threadIdx.x; i0 < n; i0 += kSortThreads * kFlight) {
    int32_t e[kFlight], blk[kFlight];
    load_entries(a, pt, hk, i0, n, e, blk);
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (blk[u] >= 0)
        a.entries[atomicAdd(&cursor[blk[u]], 1)] = e[u];
      else if (i0 + kSortThreads * u < n)
        a.part_ml[e[u]] = make_float2(-INFINITY, 0.f);
    }
  }
}

// The values' pieces stand so that the four rows of a transposing read fall
// into different banks.
template <int D>
__device__ inline int swizzle_v(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row >> 1) & 1) << 2;
}

// KT tiles of 32 keys cover the block. A wave holds 32 entries, one per lane
// pair (lane, lane ^ 32):
//   S^T[key][entry] = K . Q^T,   O^T[feature][entry] = V^T . P^T
// by 32x32x16 MFMAs; P^T goes from the first product's registers to the
// second's operand (its keys in the order 8 (u / 4) + 4 h + u % 4 of lane half
// h, which the values' reads follow). P goes as two numbers of the type, the
// rounded weight and what the rounding left: 16 bits of it in bf16, 22 in fp16,
// where one number's 8 and 11 would add as much error as the rounding of the
// result does (0.0021 against 0.0017 in bf16). m, l and the partial rows stay in
// float32. (Rows as 16-bit codes with a unit per 64 features move half the bytes
// and coarsen the features beside a large one: values with one channel of 64
// 1000 times the others' came out 0.9% off.)
// kResident workgroups share a CU, as registers and LDS let them, and the grid
// has as many: each has one item's loads under way (D 64, blocks of 64, 12 sequences
// of 350 new fp16 tokens, all of the attention: three 170 us, two 176; four would
// spill).
template <int D, int KT>
constexpr int kResident = D * KT <= 64 ? 4 : D * KT <= 128 ? 3 : 2;

template <typename T, int D, int KT>
__global__ void __launch_bounds__(256, (kResident<D, KT>)) attend_columns_kernel(ChunkArgs a) {
  using M = Unit<T>;
  using V8 = typename M::vec;
  constexpr int KEYS = 32 * KT;
  constexpr int RQ = D / 8;   // 16-byte pieces per row
  constexpr int DT = D / 32;
  // Aligned to the rows, whose bits the exclusive ors of the reads change.
  __shared__ __attribute__((aligned(256))) uint16_t Ks[KEYS * D];
  __shared__ __attribute__((aligned(256))) uint16_t Vs[KEYS * D];
  __shared__ int32_t s_ent[2][4][64];
  __shared__ int s_bad;  // the values hold infinities or NaN
  constexpr int LOADS = KEYS * RQ / 256;  // per thread, for the keys or the values
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = lane >> 5, col = lane & 31;
  const int n_items = min(*a.n_items, a.max_items);
  const uint16_t* Q = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(a.t0) * a.h_q * D;

  // A work item: where its block lies, and this lane's entry. What all lanes
  // share comes by scalar loads.
  struct Item {
    const uint16_t *k, *v;
    int count;     // entries
    int key_lim;   // keys up to the sequence's end
    int32_t pos0;  // position of the slice's first token (as if of this sequence), from the block's first key
    bool masked;   // some new token does not see all KEYS keys
    const int32_t* entries;
  };
  auto describe = [&](int item) {
    const int32_t* it = reinterpret_cast<const int32_t*>(a.items + item);
    const int32_t x = uniform_load(it), blk = uniform_load(it + 1), place = uniform_load(it + 2);
    const int32_t seq = x / a.h_kv;
    const int hk = x - seq * a.h_kv;
    const int32_t first = a.p.cu ? uniform_load(a.p.cu + seq) : seq * a.p.even;
    const int32_t end = a.p.cu ? uniform_load(a.p.cu + seq + 1) : first + a.p.even;
    const int32_t len = uniform_load(a.p.seq_lens + seq);
    int32_t page = uniform_load(a.p.table + static_cast<int64_t>(seq) * a.p.width + blk);
    page = page >= 0 && page < a.p.pages ? page : 0;
    const int64_t base = (static_cast<int64_t>(page) * a.h_kv + hk) * a.p.block * D;
    const int32_t key0 = blk * a.p.block;  // below len
    Item d;
    d.k = static_cast<const uint16_t*>(a.k) + base;
    d.v = static_cast<const uint16_t*>(a.v) + base;
    d.count = uniform_load(it + 3);
    d.key_lim = min(a.p.block, len - key0);
    d.pos0 = len - end + a.t0 - key0;
    d.masked = d.key_lim < KEYS || d.pos0 + max(first - a.t0, 0) < KEYS - 1;
    d.entries = a.entries + place;
    return d;
  };
  // Lanes' entries (the first one where a lane has none) of every other item.
  // By way of LDS: the compiler would wait for the values under way as well
  // when it copies a register that a load fills.
  auto load_entries = [&](const Item& d, int odd) {
    const int mine = wave * 32 + col;
    load_word_to_lds(d.entries + (mine < d.count ? mine : 0), &s_ent[odd][wave][0]);
  };
  // Rows past the sequence's end hold anything, their weights are 0. Rows past
  // the page (blocks that are no multiple of 32) read its last one.
  constexpr int ROWS = 256 / RQ;  // rows per load; the swizzles repeat every 16
  const int row0 = tid / RQ, piece = tid % RQ;
  const int last = a.p.block - 1;
  auto load_rows = [&](const uint16_t* src, uint16_t* dst, int swizzled) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int row = (u + 1) * ROWS > 32 * (KT - 1) ? min(row0, last - u * ROWS) : row0;
      load_to_lds(src + u * ROWS * D + (row * D + swizzled), dst + (u * 256 + wave * 64) * 8);
    }
  };
  auto load_keys = [&](const Item& d) { load_rows(d.k, Ks, 8 * (piece ^ swizzle_rows<D>(row0))); };
  auto load_values = [&](const Item& d) { load_rows(d.v, Vs, 8 * (piece ^ swizzle_v<D>(row0))); };
  V8 bq[D / 16];
  auto load_query = [&](int32_t ent) {
    const uint16_t* q = Q + static_cast<int64_t>(ent / a.slots) * D + 8 * h;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) bq[k] = __builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(q + 16 * k));
  };

  // The compiler's wait for the queries, which it makes one for every load
  // under way, falls here: before the values are asked for.
  auto have_query = [&]() {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) asm volatile("" : "+v"(bq[k]));
  };

  // LDS addresses: of the keys' operand of K-step 0, the others by exclusive or
  // (tiles 32 rows apart); of the values' of feature tile 0, likewise (steps of
  // 16 keys apart: the swizzle of a row depends on its place among 16).
  const uint32_t k_at = lds_address(&Ks[col * D + 8 * (h ^ swizzle_rows<D>(col))]);
  const int vkey = 4 * h + ((lane & 15) >> 2), vpiece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = lds_address(&Vs[vkey * D + 8 * (vpiece ^ swizzle_v<D>(vkey)) + 4 * (lane & 1)]);
  const uint32_t v_at8 =
      lds_address(&Vs[(vkey + 8) * D + 8 * (vpiece ^ swizzle_v<D>(vkey + 8)) + 4 * (lane & 1)]);

  // One item ahead: its queries and keys are on their way from when this
  // item's first product is done, its values from when the second is. The
  // entries of the one after it are asked for before those, so that the waits
  // below, which count, include them.
  int item = blockIdx.x;
  if (item >= n_items) return;
  const int stride = static_cast<int>(gridDim.x);
  Item d = describe(item), next = describe(min(item + stride, n_items - 1));
  load_entries(d, 0);
  load_entries(next, 1);
  wait_loads<0>();
  load_query(read_word(&s_ent[0][wave][lane]));
  have_query();
  load_keys(d);
  load_values(d);
  for (int odd = 0;; odd ^= 1) {
    const bool more = item + stride < n_items;
    const bool work = wave * 32 < d.count;
    const bool live = wave * 32 + col < d.count;
    const int32_t ent = read_word(&s_ent[odd][wave][lane]);
    const int lim = live ? min(d.key_lim - 1, d.pos0 + ent / a.slots / a.h_q) : -1;  // last key seen
    wait_loads<LOADS>();  // all but the values
    meet();
    if (tid == 0) s_bad = 0;
    floatx16_t s[KT];
    if (work) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = floatx16_t{};
      auto step = [&](auto kc) {
        constexpr int k = decltype(kc)::value;
        u32x4 x[KT];
        read_rows<32 * k, 32 * D * 2>(k_at, x);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = M::mma(__builtin_bit_cast(V8, x[kt]), bq[k], s[kt]);
      };
      steps(std::make_integer_sequence<int, D / 16>{}, step);
    }
    meet();  // every wave is done with the keys
    Item after = next;
    if (more) {
      after = describe(min(item + 2 * stride, n_items - 1));
      load_query(read_word(&s_ent[odd ^ 1][wave][lane]));
      load_entries(after, odd);
      load_keys(next);
    }
    const bool whole = __all(!live || lim == KEYS - 1);
    float m = -INFINITY, l = 0.f;
    V8 bp[KEYS / 16], bl[KEYS / 16];
    if (work) {
      // s[kt][v] is key 32 kt + 8 (v / 4) + 4 h + v % 4.
      if (!whole) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int key = kt * 32 + 8 * (v >> 2) + 4 * h + (v & 3);
            s[kt][v] = key <= lim ? s[kt][v] : -INFINITY;
          }
      }
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) m = fmaxf(m, s[kt][v]);
      m = fmaxf(m, __shfl_xor(m, 32));
      const float mz = m > -INFINITY ? m : 0.f;
      m = m * a.scale_log2 - M::kShift;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          // The difference first: at most 2^kShift however large the scores are.
          const float p = __builtin_amdgcn_exp2f(fmaf(s[kt][v] - mz, a.scale_log2, M::kShift));
          s[kt][v] = p;
          l += p;
        }
      l += __shfl_xor(l, 32);
#pragma unroll
      for (int j = 0; j < KEYS / 16; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float p = s[j >> 1][8 * (j & 1) + u];
          bp[j][u] = static_cast<typename M::scalar>(p);
          bl[j][u] = static_cast<typename M::scalar>(p - static_cast<float>(bp[j][u]));
        }
    }
    if (more)
      wait_loads<LOADS>();  // all but the next keys
    else
      wait_loads<0>();
    meet();
    // A weight of 0 times an infinite or NaN value is NaN, but a value that a
    // query does not see must not reach it. Where the block has hidden keys,
    // such values are taken out, and put back after the product for the
    // queries that see them.
    bool bad = false;
    if (d.masked) {
      u32x4 x[LOADS];
#pragma unroll
      for (int u = 0; u < LOADS; ++u) x[u] = *reinterpret_cast<const u32x4*>(&Vs[(u * 256 + tid) * 8]);
      uint32_t found = 0;
#pragma unroll
      for (int u = 0; u < LOADS; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          found |= (x[u][w] & M::kInf) == M::kInf ? 1u : 0u;
          found |= ((x[u][w] >> 16) & M::kInf) == M::kInf ? 1u : 0u;
        }
      if (found) s_bad = 1;
      meet();
      bad = s_bad != 0;
      if (bad) {
        for (int i = tid * 8; i < KEYS * D; i += 256 * 8)
          for (int e = 0; e < 8; ++e)
            if ((Vs[i + e] & M::kInf) == M::kInf) Vs[i + e] = 0;
        meet();
      }
    }
    // Two feature tiles at a time.
    if (work) {
      if (live && h == 0) a.part_ml[ent] = make_float2(m, l);
      auto half = [&](auto pc) {
        constexpr int dt = 2 * decltype(pc)::value;
        floatx16_t o[2] = {floatx16_t{}, floatx16_t{}};
        // Features 32 dt + [0, 64), keys 16 j + [0, 16).
        auto step = [&](auto jc) {
          constexpr int j = decltype(jc)::value;
          u32x2 x[4];
          read_transposed<64 * dt, j * 16 * D * 2>(v_at, v_at8, x);
          const V8 y[2] = {__builtin_bit_cast(V8, u32x4{x[0][0], x[0][1], x[1][0], x[1][1]}),
                           __builtin_bit_cast(V8, u32x4{x[2][0], x[2][1], x[3][0], x[3][1]})};
#pragma unroll
          for (int t = 0; t < 2; ++t) o[t] = M::mma(y[t], bp[j], o[t]);
#pragma unroll
          for (int t = 0; t < 2; ++t) o[t] = M::mma(y[t], bl[j], o[t]);
        };
        steps(std::make_integer_sequence<int, KEYS / 16>{}, step);
        // The second parts of weights, zeros and negative numbers among them,
        // make NaN of an infinite value.
        uint32_t lost = 0;
        if (!d.masked) {
          float z = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) z = fmaf(o[e / 16][e % 16], 0.f, z);
          if (__any(z != z)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = o[e / 16][e % 16];
              lost |= x != x ? 1u << e : 0u;
              o[e / 16][e % 16] = x != x ? 0.f : x;
            }
          }
        }
        const bool again = __any(lost);
        if (bad || again) {
          // What the queries see of the values that were taken out or lost.
          for (int key = 0; key < d.key_lim; ++key) {
            const uint16_t* row = d.v + key * D + 32 * dt + 4 * h;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(row + t * 32 + 8 * q4);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                  const uint16_t bits = static_cast<uint16_t>(x[w >> 1] >> (16 * (w & 1)));
                  if ((bits & M::kInf) == M::kInf && key <= lim)
                    o[t][4 * q4 + w] += static_cast<float>(__builtin_bit_cast(typename M::scalar, bits));
                }
              }
          }
        }
        if (again) {  // sums of finite values that left the range
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float x = o[e / 16][e % 16];
            o[e / 16][e % 16] = (lost >> e) & 1u && x == 0.f ? NAN : x;
          }
        }
        if (live) {
          float* dst = a.part_acc + static_cast<int64_t>(ent) * D + 32 * dt + 4 * h;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
              *reinterpret_cast<float4*>(dst + t * 32 + 8 * q4) =
                  make_float4(o[t][4 * q4], o[t][4 * q4 + 1], o[t][4 * q4 + 2], o[t][4 * q4 + 3]);
        }
      };
      steps(std::make_integer_sequence<int, DT / 2>{}, half);
    }
    have_query();
    meet();  // every wave is done with the values
    if (!more) break;
    load_values(next);
    d = next;
    next = after;
    item += stride;
  }
}

// One workgroup per token: each query head's slots merged by D / 8 lanes.
template <typename T, int D>
__global__ void __launch_bounds__(512) merge_slots_kernel(ChunkArgs a) {
  constexpr int LPR = D / 8;
  const int32_t tok = a.t0 + blockIdx.x;
  if (locate(a.p, tok).pos < 0) return;
  const int c = threadIdx.x % LPR;
  for (int hd = threadIdx.x / LPR; hd < a.h_q; hd += blockDim.x / LPR) {
    const int64_t e0 = (static_cast<int64_t>(blockIdx.x) * a.h_q + hd) * a.slots;
    const float2* ml = a.part_ml + e0;
    const float4* acc = reinterpret_cast<const float4*>(a.part_acc + e0 * D) + 2 * c;
    // Eight slots in flight. Those that were not written (m = -inf, l = 0) hold
    // anything: they count as zeros. Where every score is NaN, m is -inf too (a
    // maximum leaves NaN out) and l is NaN: the slot counts.
    float top = -INFINITY, total = 0.f, o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
    for (int j0 = 0; j0 < a.slots; j0 += 8) {
      float2 x[8];
      float4 raw[8][2];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = min(j0 + u, a.slots - 1);
        x[u] = ml[j];
        raw[u][0] = acc[j * (D / 4)];
        raw[u][1] = acc[j * (D / 4) + 1];
      }
      float m = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (j0 + u >= a.slots) x[u] = make_float2(-INFINITY, 0.f);
        m = fmaxf(m, x[u].x);
      }
      const float z = m > -INFINITY ? m : 0.f;
      const float old = __builtin_amdgcn_exp2f(top - z);
      total *= old;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= old;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const bool in = x[u].x != -INFINITY || x[u].y != 0.f;
        const float w = __builtin_amdgcn_exp2f(x[u].x - z);
        total = fmaf(x[u].y, w, total);
        const float v[8] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w,
                            raw[u][1].x, raw[u][1].y, raw[u][1].z, raw[u][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(in ? v[e] : 0.f, w, o[e]);
      }
      top = m;
    }
    const int64_t row = static_cast<int64_t>(tok) * a.h_q + hd;
    T* out = static_cast<T*>(a.out) + row * D + 8 * c;
    T y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      Elem<T>::store(y, e, total > 0.f ? o[e] / total : (total == 0.f ? 0.f : o[e] + total));
    *reinterpret_cast<u32x4*>(out) = __builtin_bit_cast(u32x4, y);
    if (a.lse && c == 0)
      a.lse[hd * static_cast<int64_t>(a.p.tokens) + tok] =
          total > 0.f ? top + log2f(total) : (total == 0.f ? -INFINITY : total);
  }
}

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

// Block by block pays where an entry's block is on average another's too, and
// where the entries' keys and values, which rows read one by one, outweigh the
// launches. bf16, 32 and 8 heads of 128, 9 blocks of 128 per query, whole calls
// block by block and row by row: 32 sequences of 256 blocks, 4 new tokens each
// (0.6 entries per block) 413 and 314 us, 8 each (1.1) 631 and 577, 16 each (2.2)
// 855 and 1102; one of 512 blocks, 8 tokens 65 and 27, 32 tokens (0.6 GB) 88 and
// 77, 64 tokens (1.2 GB) 98 and 145. 8 heads of 64, 5 blocks of 64: 8 of 64 blocks,
// 64 tokens each (335 MB) 43 and 32, 128 tokens each (671 MB) 49 and 58.
constexpr int64_t kColumnBytes = int64_t(1) << 29;
bool chunk_takes(const moba_paged& c) {
  const int64_t entries = c.tokens * c.h_q * c.slots;
  return c.dtype != MOBA_FP32 && (c.head_dim == 64 || c.head_dim == 128) && c.block_size <= 128 &&
         c.table_width <= 15360 && c.h_kv <= 65535 && 2 * entries >= 3 * c.seqs * c.h_kv * c.table_width &&
         entries * c.block_size * c.head_dim * 4 >= kColumnBytes;
}

ChunkPlan chunk_plan(const moba_paged& c) {
  ChunkPlan pl;
  const int64_t per_token = c.h_q * c.slots;
  // Partial rows of at most 2^29 bytes at a time.
  pl.slice = (int64_t(1) << 29) / (per_token * c.head_dim * 4);
  pl.slice = pl.slice < 1 ? 1 : (pl.slice < c.tokens ? pl.slice : c.tokens);
  // Parts of 64 tokens: more workgroups count and place, and the scan walks more
  // parts (4 x 512 tokens, 4 kv heads: the attention 224 us, in parts of 256
  // 255; 2048 tokens, 8 kv heads: 307 and 308). Longer ones where a slice has
  // more than 64 of them or the count table would pass 2^22 entries.
  pl.part = 64;
  while (pl.slice / pl.part > 64) pl.part *= 2;
  const int64_t row = c.h_kv * c.table_width;
  while (pl.part < pl.slice && (pl.slice / pl.part + c.seqs) * row > (int64_t(1) << 22)) pl.part *= 2;
  pl.parts = cdiv(pl.slice, pl.part) + c.seqs;
  const int64_t entries = pl.slice * per_token;
  const int64_t items = cdiv(entries, kItem) + c.seqs * row;
  pl.max_items = items < entries ? items : entries;
  size_t o = 256;
  auto take = [&](size_t bytes) { const size_t at = o; o += up256(bytes); return at; };
  pl.table = take(sizeof(int32_t) * static_cast<size_t>(pl.parts * row));
  pl.items = take(sizeof(int4) * static_cast<size_t>(pl.max_items));
  pl.entries = take(sizeof(int32_t) * static_cast<size_t>(entries));
  pl.ml = take(sizeof(float2) * static_cast<size_t>(entries));
  pl.acc = take(sizeof(float) * static_cast<size_t>(entries * c.head_dim));
  pl.total = o;
  return pl;
}

int chunk_attend(const moba_paged& c, const Paged& p, void* workspace, hipStream_t s) {
  const ChunkPlan pl = chunk_plan(c);
  char* ws = static_cast<char*>(workspace);
  ChunkArgs a;
  a.p = p;
  a.q = c.q;
  a.k = c.k;
  a.v = c.v;
  a.block_idx = c.block_idx;
  a.out = c.out;
  a.lse = c.lse;
  a.n_items = reinterpret_cast<int32_t*>(ws);
  a.table = reinterpret_cast<int32_t*>(ws + pl.table);
  a.items = reinterpret_cast<int4*>(ws + pl.items);
  a.entries = reinterpret_cast<int32_t*>(ws + pl.entries);
  a.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
  a.part_acc = reinterpret_cast<float*>(ws + pl.acc);
  a.h_q = static_cast<int>(c.h_q);
  a.h_kv = static_cast<int>(c.h_kv);
  a.slots = static_cast<int>(c.slots);
  a.part = static_cast<int>(pl.part);
  a.parts = static_cast<int>(pl.parts);
  a.max_items = static_cast<int>(pl.max_items);
  a.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(c.head_dim)));
  const dim3 parts(static_cast<unsigned>(pl.parts), static_cast<unsigned>(c.h_kv));
  const unsigned lds = static_cast<unsigned>(sizeof(int32_t) * c.table_width);
  for (int64_t t0 = 0; t0 < c.tokens; t0 += pl.slice) {
    a.t0 = static_cast<int32_t>(t0);
    a.t1 = static_cast<int32_t>(c.tokens - t0 < pl.slice ? c.tokens : t0 + pl.slice);
    hipLaunchKernelGGL(column_count_kernel, parts, dim3(kSortThreads), lds, s, a);
    hipLaunchKernelGGL(column_scan_kernel, dim3(static_cast<unsigned>(c.seqs), static_cast<unsigned>(c.h_kv)),
                       dim3(1024), lds, s, a);
    hipLaunchKernelGGL(column_place_kernel, parts, dim3(kSortThreads), lds, s, a);
    int st = check_launch("moba_paged_attend (columns)");
    if (st) return st;
    auto attend = [&](auto t, auto dim, auto kt) {
      using T = decltype(t);
      constexpr int D = decltype(dim)::value, KT = decltype(kt)::value;
      constexpr int64_t kGrid = 256 * kResident<D, KT>;
      const int64_t most = pl.max_items < kGrid ? pl.max_items : kGrid;
      hipLaunchKernelGGL((attend_columns_kernel<T, D, KT>), dim3(static_cast<unsigned>(most)), dim3(256), 0, s, a);
      int rc = check_launch("moba_paged_attend (attend)");
      if (rc) return rc;
      const int64_t lanes = c.h_q * (D / 8);
      hipLaunchKernelGGL((merge_slots_kernel<T, D>), dim3(static_cast<unsigned>(a.t1 - a.t0)),
                         dim3(lanes <= 64 ? 64 : lanes <= 128 ? 128 : lanes <= 256 ? 256 : 512), 0, s, a);
      return check_launch("moba_paged_attend (merge)");
    };
    auto tiles = [&](auto t, auto dim) {
      if (c.block_size <= 32) return attend(t, dim, std::integral_constant<int, 1>{});
      if (c.block_size <= 64) return attend(t, dim, std::integral_constant<int, 2>{});
      if (c.block_size <= 96) return attend(t, dim, std::integral_constant<int, 3>{});
      return attend(t, dim, std::integral_constant<int, 4>{});
    };
    auto dims = [&](auto t) {
      if (c.head_dim == 64) return tiles(t, std::integral_constant<int, 64>{});
      return tiles(t, std::integral_constant<int, 128>{});
    };
    st = c.dtype == MOBA_BF16 ? dims(bf16_t{}) : dims(f16_t{});
    if (st) return st;
  }
  return MOBA_OK;
}

}  // namespace moba
