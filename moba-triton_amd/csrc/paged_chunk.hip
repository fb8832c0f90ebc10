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
// An entry is its index in block_idx, which is also the index of its partial
// row. Entries of a column stand in no particular order; nothing depends on it.
#include "paged_chunk.h"

#include "paged_gate.h"

namespace moba {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Unit;
template <> struct Unit<bf16_t> {
  typedef bf16x8_t vec;
  typedef __bf16 scalar;
  static constexpr uint32_t kInf = 0x7f80u;
  __device__ static floatx16_t mma(vec a, vec b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Unit<f16_t> {
  typedef f16x8_t vec;
  typedef _Float16 scalar;
  static constexpr uint32_t kInf = 0x7c00u;
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

// counts[part, kv head, block]; dynamic LDS: width counters. grid (parts, h_kv).
__global__ void __launch_bounds__(256) column_count_kernel(ChunkArgs a) {
  extern __shared__ int32_t bins[];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.n_items = 0;
  const Part pt = find_part(a.p, a.t0, a.t1, a.part, blockIdx.x);
  if (pt.seq < 0) return;
  const int hk = blockIdx.y, group = a.h_q / a.h_kv, per = group * a.slots;
  for (int j = threadIdx.x; j < a.p.width; j += 256) bins[j] = 0;
  __syncthreads();
  const int n = (pt.end - pt.begin) * per;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int64_t e = (static_cast<int64_t>(pt.begin + i / per) * a.h_q + hk * group) * a.slots + i % per;
    const int32_t blk = entry_block(a.p, pt.seq, a.block_idx[e]);
    if (blk >= 0) atomicAdd(&bins[blk], 1);
  }
  __syncthreads();
  int32_t* out = a.table + (static_cast<int64_t>(blockIdx.x) * a.h_kv + hk) * a.p.width;
  for (int j = threadIdx.x; j < a.p.width; j += 256) out[j] = bins[j];
}

// Per (sequence, kv head): table -> the place of every (part, block)'s first
// entry; work items of the columns. grid (seqs, h_kv).
__global__ void __launch_bounds__(1024) column_scan_kernel(ChunkArgs a) {
  __shared__ int32_t wsum[2][16];
  __shared__ int32_t base_item;
  const int32_t seq = blockIdx.x;
  const int hk = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // This sequence's parts and where its entries begin.
  const NewTokens r = new_tokens(a.p, seq);
  const int32_t lo = max(r.first, a.t0), hi = min(r.first + r.n, a.t1);
  if (hi <= lo) return;
  int32_t first = 0;
  for (int32_t base = 0; base < seq; base += 64) {
    int32_t mine = 0;
    if (base + lane < seq) {
      const NewTokens o = new_tokens(a.p, base + lane);
      const int32_t l = max(o.first, a.t0), h = min(o.first + o.n, a.t1);
      mine = h > l ? (h - l + a.part - 1) / a.part : 0;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) mine += __shfl_xor(mine, off);
    first += mine;
  }
  const int32_t parts = (hi - lo + a.part - 1) / a.part;
  if (first + parts > a.parts) return;  // only where sequences claim the same tokens
  const int per = a.h_q / a.h_kv * a.slots;
  const int32_t place0 = (lo - a.t0) * a.h_q * a.slots + hk * (hi - lo) * per;
  const int64_t row = static_cast<int64_t>(a.h_kv) * a.p.width;
  int32_t* table = a.table + static_cast<int64_t>(first) * row + static_cast<int64_t>(hk) * a.p.width;
  const int32_t blocks = min(a.p.width, (r.len + a.p.block - 1) / a.p.block);
  // Two rounds over the columns: the number of items, then the lists.
  int32_t items = 0;
  for (int round = 0; round < 2; ++round) {
    int32_t carry_e = 0, carry_i = 0;
    for (int32_t b0 = 0; b0 < blocks; b0 += 1024) {
      const int32_t b = b0 + threadIdx.x;
      int32_t n = 0;
      if (b < blocks) {
        for (int32_t q = 0; q < parts; ++q) n += table[q * row + b];
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
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        if (w < wave) { ie += wsum[0][w]; ii += wsum[1][w]; }
        te += wsum[0][w];
        ti += wsum[1][w];
      }
      __syncthreads();
      if (round == 1 && b < blocks) {
        int32_t at = place0 + carry_e + ie - n;
        const int32_t start = at;
        for (int32_t q = 0; q < parts; ++q) {
          const int32_t c = table[q * row + b];
          table[q * row + b] = at;
          at += c;
        }
        const int32_t i0 = base_item + carry_i + ii - k;
        for (int32_t i = 0; i < k && i0 + i < a.max_items; ++i)
          a.items[i0 + i] = make_int4(seq * a.h_kv + hk, b, start + i * kItem, min(kItem, n - i * kItem));
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
__global__ void __launch_bounds__(256) column_place_kernel(ChunkArgs a) {
  extern __shared__ int32_t cursor[];
  const Part pt = find_part(a.p, a.t0, a.t1, a.part, blockIdx.x);
  if (pt.seq < 0) return;
  const int hk = blockIdx.y, group = a.h_q / a.h_kv, per = group * a.slots;
  const int32_t* row = a.table + (static_cast<int64_t>(blockIdx.x) * a.h_kv + hk) * a.p.width;
  for (int j = threadIdx.x; j < a.p.width; j += 256) cursor[j] = row[j];
  __syncthreads();
  const int n = (pt.end - pt.begin) * per;
  const int64_t e0 = static_cast<int64_t>(a.t0) * a.h_q * a.slots;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int64_t e = (static_cast<int64_t>(pt.begin + i / per) * a.h_q + hk * group) * a.slots + i % per;
    const int32_t blk = entry_block(a.p, pt.seq, a.block_idx[e]);
    if (blk >= 0)
      a.entries[atomicAdd(&cursor[blk], 1)] = static_cast<int32_t>(e - e0);
    else
      *reinterpret_cast<float2*>(a.part_ml + 2 * (e - e0)) = make_float2(-INFINITY, 0.f);
  }
}

// 16-byte pieces of a row stand in LDS at piece ^ swizzle(row), so that the 16
// rows a wave's lanes read together (keys), or the four rows of a transposing
// read (values), fall into different banks.
template <int D>
__device__ inline int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ inline int swizzle_v(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row >> 1) & 1) << 2;
}

// Eight elements of V^T for one MFMA operand: two transposing reads
// (ds_read_b64_tr_b16), each of four keys by 16 features per 16 lanes.
typedef short v4i16_t __attribute__((ext_vector_type(4)));
template <typename V>
__device__ inline V transposed(const uint16_t* p0, const uint16_t* p1) {
  typedef __attribute__((address_space(3))) v4i16_t lds_v4i16;
  const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p0));
  const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p1));
  typedef short v8i16_t __attribute__((ext_vector_type(8)));
  const v8i16_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(V, v);
}

// 16 bytes from global memory straight to LDS: lane i's to `dst` + 16 i.
__device__ inline void load_to_lds(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(src)),
      (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// KT tiles of 32 keys cover the block. A wave holds 32 entries, one per lane
// pair (lane, lane ^ 32):
//   S^T[key][entry] = K . Q^T,   O^T[feature][entry] = V^T . P^T
// by 32x32x16 MFMAs; P^T goes from the first product's registers to the
// second's operand (its keys in the order 8 (u / 4) + 4 h + u % 4 of lane half
// h, which the values' reads follow). P is rounded to the type for the
// product, as the framework's forward does; m and l stay in float32. Partial
// rows are rounded to the type once: their weighted mean moves by at most half
// a step of the weighted mean of |v|.
template <typename T, int D, int KT>
__global__ void __launch_bounds__(256, 2) attend_columns_kernel(ChunkArgs a) {
  using M = Unit<T>;
  using V8 = typename M::vec;
  constexpr int KEYS = 32 * KT;
  constexpr int RQ = D / 8;   // 16-byte pieces per row
  constexpr int DT = D / 32;
  __shared__ __attribute__((aligned(16))) uint16_t Ks[KEYS * D];
  __shared__ __attribute__((aligned(16))) uint16_t Vs[KEYS * D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = lane >> 5, col = lane & 31;
  const int n_items = min(*a.n_items, a.max_items);
  const uint16_t* Q = static_cast<const uint16_t*>(a.q) + static_cast<int64_t>(a.t0) * a.h_q * D;
  for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
    const int4 it = a.items[item];
    const int32_t seq = it.x / a.h_kv;
    const int hk = it.x - seq * a.h_kv;
    const NewTokens nt = new_tokens(a.p, seq);
    const int64_t key0 = static_cast<int64_t>(it.y) * a.p.block;
    const int key_lim = static_cast<int>(min(static_cast<int64_t>(a.p.block), nt.len - key0));
    const int32_t page = max(page_of(a.p, seq, it.y), 0);
    const int64_t base = (static_cast<int64_t>(page) * a.h_kv + hk) * a.p.block * D;
    const uint16_t* kg = static_cast<const uint16_t*>(a.k) + base;
    const uint16_t* vg = static_cast<const uint16_t*>(a.v) + base;
    // Rows past the sequence's end read its last one; their weights are 0.
#pragma unroll
    for (int u = 0; u < KEYS * RQ / 256; ++u) {
      const int i = u * 256 + tid, row = i / RQ, piece = i % RQ;
      load_to_lds(kg + min(row, key_lim - 1) * D + 8 * (piece ^ swizzle_k<D>(row)),
                  &Ks[(u * 256 + wave * 64) * 8]);
    }
#pragma unroll
    for (int u = 0; u < KEYS * RQ / 256; ++u) {
      const int i = u * 256 + tid, row = i / RQ, piece = i % RQ;
      load_to_lds(vg + min(row, key_lim - 1) * D + 8 * (piece ^ swizzle_v<D>(row)),
                  &Vs[(u * 256 + wave * 64) * 8]);
    }
    const int mine = wave * 32 + col;
    const bool live = mine < it.w;
    const int32_t ent = a.entries[it.z + (live ? mine : 0)];
    const int32_t qrow = ent / a.slots;
    V8 bq[D / 16];
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
      bq[k] = __builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(
                                         Q + static_cast<int64_t>(qrow) * D + 16 * k + 8 * h));
    const int32_t pos = nt.len - nt.n + (a.t0 + qrow / a.h_q - nt.first);
    const int64_t row_lim = pos - key0;
    const int lim = live ? static_cast<int>(min(static_cast<int64_t>(key_lim - 1), row_lim)) : -1;
    // Loads to LDS count as vector memory: a barrier alone does not wait for them.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (wave * 32 < it.w) {
      floatx16_t s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = floatx16_t{};
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int row = kt * 32 + col;
          const V8 ka = __builtin_bit_cast(V8, *reinterpret_cast<const u32x4*>(
                                                   &Ks[row * D + 8 * ((2 * k + h) ^ swizzle_k<D>(row))]));
          s[kt] = M::mma(ka, bq[k], s[kt]);
        }
      // s[kt][v] is key 32 kt + 8 (v / 4) + 4 h + v % 4.
      const bool whole = __all(!live || lim == KEYS - 1);
      float m = -INFINITY, l = 0.f;
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
      m = fmaxf(m, __shfl_xor(m, 32)) * a.scale_log2;
      const float mz = m > -INFINITY ? m : 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[kt][v], a.scale_log2, -mz));
          s[kt][v] = p;
          l += p;
        }
      l += __shfl_xor(l, 32);
      V8 bp[KEYS / 16];
#pragma unroll
      for (int j = 0; j < KEYS / 16; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u)
          bp[j][u] = static_cast<typename M::scalar>(s[j >> 1][8 * (j & 1) + u]);
      // Value operand of features 32 dt + [0, 32) and keys 16 j + [0, 16).
      auto values = [&](int j, int dt) {
        const int key = 16 * j + 4 * h + ((lane & 15) >> 2);
        const int piece = dt * 4 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        const uint16_t* p0 = &Vs[key * D + 8 * (piece ^ swizzle_v<D>(key)) + 4 * (lane & 1)];
        const uint16_t* p1 = &Vs[(key + 8) * D + 8 * (piece ^ swizzle_v<D>(key + 8)) + 4 * (lane & 1)];
        return transposed<V8>(p0, p1);
      };
      floatx16_t o[DT];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = floatx16_t{};
#pragma unroll
      for (int j = 0; j < KEYS / 16; ++j)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = M::mma(values(j, dt), bp[j], o[dt]);
      if (!whole) {
        // A weight of 0 times an infinite or NaN value is NaN, but a value
        // that a query does not see must not reach it. Where any result is
        // not finite: the product again without such values, and who sees
        // which of them by two more products of zeros and ones.
        float bad = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; ++v) bad = fmaf(o[dt][v], 0.f, bad);
        if (__any(bad != 0.f)) {
          using S = typename M::scalar;
          for (int dt = 0; dt < DT; ++dt) {
            floatx16_t fin = floatx16_t{}, up = floatx16_t{}, down = floatx16_t{};
#pragma unroll
            for (int j = 0; j < KEYS / 16; ++j) {
              const V8 va = values(j, dt);
              V8 f, pu, nu, see;
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const uint32_t bits = __builtin_bit_cast(uint16_t, va[u]);
                const bool inf = (bits & 0x7fffu) == M::kInf, nan = (bits & 0x7fffu) > M::kInf;
                f[u] = inf || nan ? static_cast<S>(0.f) : va[u];
                pu[u] = static_cast<S>(nan || (inf && !(bits & 0x8000u)) ? 1.f : 0.f);
                nu[u] = static_cast<S>(nan || (inf && (bits & 0x8000u)) ? 1.f : 0.f);
                const int key = 16 * j + 8 * (u >> 2) + 4 * h + (u & 3);
                see[u] = static_cast<S>(key <= lim ? 1.f : 0.f);
              }
              fin = M::mma(f, bp[j], fin);
              up = M::mma(pu, see, up);
              down = M::mma(nu, see, down);
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const float x = up[v] > 0.f ? INFINITY : 0.f, y = down[v] > 0.f ? INFINITY : 0.f;
              fin[v] += x - y;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
              if (d == dt) o[d] = fin;
          }
        }
      }
      if (live) {
        if (h == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * static_cast<int64_t>(ent)) = make_float2(m, l);
        uint16_t* dst = static_cast<uint16_t*>(a.part_acc) + static_cast<int64_t>(ent) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            typedef typename M::scalar S4 __attribute__((ext_vector_type(4)));
            S4 x;
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] = static_cast<typename M::scalar>(o[dt][4 * q4 + w]);
            *reinterpret_cast<u32x2*>(dst + dt * 32 + 8 * q4) = __builtin_bit_cast(u32x2, x);
          }
      }
    }
    __syncthreads();  // every wave is done with the staged rows
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
    const float* ml = a.part_ml + 2 * e0;
    const u32x4* acc = static_cast<const u32x4*>(a.part_acc) + e0 * LPR + c;
    float top = -INFINITY;
    for (int j = 0; j < a.slots; ++j) top = fmaxf(top, ml[2 * j]);
    const float z = top > -INFINITY ? top : 0.f;
    float total = 0.f, o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
    for (int j = 0; j < a.slots; ++j) {
      const float m = ml[2 * j];
      if (m == -INFINITY) continue;  // nothing was written there
      const float w = __builtin_amdgcn_exp2f(m - z);
      total = fmaf(ml[2 * j + 1], w, total);
      const u32x4 raw = acc[j * LPR];
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(Elem<T>::load(x, e), w, o[e]);
    }
    const int64_t row = static_cast<int64_t>(tok) * a.h_q + hd;
    T* out = static_cast<T*>(a.out) + row * D + 8 * c;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      Elem<T>::store(out, e, total > 0.f ? o[e] / total : (total == 0.f ? 0.f : o[e] + total));
    if (a.lse && c == 0)
      a.lse[hd * static_cast<int64_t>(a.p.tokens) + tok] =
          total > 0.f ? top + log2f(total) : (total == 0.f ? -INFINITY : total);
  }
}

size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

bool chunk_takes(const moba_paged& c) {
  return c.dtype != MOBA_FP32 && (c.head_dim == 64 || c.head_dim == 128) && c.block_size <= 128 &&
         c.table_width <= 16384 && c.h_kv <= 65535 && c.tokens >= 4 * c.seqs;
}

ChunkPlan chunk_plan(const moba_paged& c) {
  ChunkPlan pl;
  const int64_t per_token = c.h_q * c.slots;
  // Partial rows of at most 2^29 bytes at a time.
  pl.slice = (int64_t(1) << 29) / (per_token * c.head_dim * 2);
  pl.slice = pl.slice < 1 ? 1 : (pl.slice < c.tokens ? pl.slice : c.tokens);
  // Parts of 64 tokens, more where the count table would pass 2^22 entries.
  pl.part = 64;
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
  pl.ml = take(sizeof(float) * 2 * static_cast<size_t>(entries));
  pl.acc = take(2 * static_cast<size_t>(entries * c.head_dim));
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
  a.part_ml = reinterpret_cast<float*>(ws + pl.ml);
  a.part_acc = ws + pl.acc;
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
    hipLaunchKernelGGL(column_count_kernel, parts, dim3(256), lds, s, a);
    hipLaunchKernelGGL(column_scan_kernel, dim3(static_cast<unsigned>(c.seqs), static_cast<unsigned>(c.h_kv)),
                       dim3(1024), 0, s, a);
    hipLaunchKernelGGL(column_place_kernel, parts, dim3(256), lds, s, a);
    int st = check_launch("moba_paged_attend (columns)");
    if (st) return st;
    auto attend = [&](auto t, auto dim, auto kt) {
      using T = decltype(t);
      constexpr int D = decltype(dim)::value, KT = decltype(kt)::value;
      const int64_t most = pl.max_items < 512 ? pl.max_items : 512;
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
