// MoBA attention of new tokens over a paged cache: softmax(q . k / sqrt D) v
// over the keys, up to the token's own position, of the blocks that
// paged_gate.hip chose. Here each query by itself, every type and size;
// paged_chunk.hip goes block by block where many queries share blocks.
#include "paged.h"
#include "paged_chunk.h"
#include "paged_gate.h"
#include "rotary.h"

namespace moba {

namespace {

struct RowArgs {
  Paged p;
  const void* q;             // [tokens, h_q, D]
  const void* k;             // pages
  const void* v;
  const int32_t* block_idx;  // [tokens, h_q, slots], or null: chosen here from
  const uint32_t* keys;      // the scores [tokens, h_q, width]
  void* out;                 // [tokens, h_q, D]
  float* lse;                // [h_q, tokens] log2 units, or null
  float* part_ml;            // [rows, splits, 2]
  float* part_o;             // [rows, splits, D]
  int64_t row0;              // first row of this launch
  int h_q, h_kv, slots, splits;
  int take, current;
  float scale_log2;
};

// A row's result from its maximum (log2 units), sum and weighted values. No
// visible key: 0, lse -inf; a sum that is not a number stays one.
__device__ inline float row_value(float x, float total) {
  return total > 0.f ? x / total : (total == 0.f ? 0.f : x + total);
}
__device__ inline float row_lse(float top, float total) {
  return total > 0.f ? top + log2f(total) : (total == 0.f ? -INFINITY : total);
}

// One query head of one token per workgroup (and split): its chosen blocks in
// runs of 64 / LPR * U keys, one run after another per wave. D / F lanes share
// a key, F features each; every lane group keeps its own running maximum and
// sum, and they meet at the end. All in float32.
//
// TM > 0: the blocks are chosen here, from the scores, by all waves: every
// lane the best of every 64 NW-th score, every wave the best of its lanes, the
// first wave the best of the waves (as select_kernel, without its launch and
// its trip through memory).
//
// Memory-bound with many rows: one token of each of 32 sequences of up to 100k
// keys, 32 and 8 heads of 128 in bf16, 8 blocks of 128 each: 96 us, 118 with the
// scores, where the bytes of both take 94 at the rate of a large copy. One
// sequence with 4 heads of 64 over 64k keys: 11 us, the latency of choosing
// and of one pass.
template <typename T, int D, int NW, int TM>
__global__ void __launch_bounds__(64 * NW) attend_rows_kernel(RowArgs a) {
  constexpr int F = 16 / static_cast<int>(sizeof(T));
  constexpr int LPR = D / F;
  constexpr int RPW = 64 / LPR;  // keys per load instruction
  constexpr int U = 8;
  constexpr int KEYS = RPW * U;
  constexpr int TS = TM ? TM : 1;
  using Best = WaveBest<Rank<T>, TS>;
  __shared__ float s_o[NW][D];
  __shared__ float s_m[NW], s_l[NW];
  __shared__ typename Best::Word s_best[NW][TS];
  __shared__ int32_t s_ids[TS + 1];
  const int64_t row = a.row0 + blockIdx.x;
  const int32_t tok = static_cast<int32_t>(row / a.h_q);
  const int h = static_cast<int>(row % a.h_q);
  const int hk = h / (a.h_q / a.h_kv);
  const TokenAt at = locate(a.p, tok);
  if (at.pos < 0) return;  // its rows stay as they were
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane % LPR, g = lane / LPR;
  const int bs = a.p.block;
  float q[F];
  {
    const T* qp = static_cast<const T*>(a.q) + row * D + c * F;
#pragma unroll
    for (int e = 0; e < F; ++e) q[e] = Elem<T>::load(qp, e) * a.scale_log2;
  }
  const int32_t* ids = TM ? s_ids : a.block_idx + row * a.slots;
  if constexpr (TM > 0) {
    const int32_t own = at.pos / bs;
    const int32_t past = a.take ? min(own, a.p.width) : 0;
    Best list;
    list.clear();
    list.add_all(a.keys + row * a.p.width, past, wave * 64 + lane, 64 * NW);
    list.meet();
    if (lane < TM) s_best[wave][lane] = list.mine();
    __syncthreads();
    if (wave == 0) {
      list.clear();
#pragma unroll
      for (int i = 0; i < NW * TM; i += 64)
        if (i + lane < NW * TM) list.add((&s_best[0][0])[i + lane]);
      list.meet();
      list.emit(a.take, own_entry(a.p, a.current, at.seq, own), a.slots, s_ids);
    }
    __syncthreads();
  }
  float m = -INFINITY, l = 0.f, o[F];
#pragma unroll
  for (int e = 0; e < F; ++e) o[e] = 0.f;
  const int per_block = (bs + KEYS - 1) / KEYS;
  const int units = a.slots * per_block;
  for (int u = blockIdx.y * NW + wave; u < units; u += a.splits * NW) {
    const int32_t blk = ids[u / per_block];
    if (blk < 0) continue;
    const int32_t page = page_of(a.p, at.seq, blk);
    if (page < 0) continue;
    const int64_t seen64 = static_cast<int64_t>(at.pos) - static_cast<int64_t>(blk) * bs + 1;
    const int seen = seen64 < bs ? static_cast<int>(seen64) : bs;  // visible keys of the block
    const int k0 = (u % per_block) * KEYS;
    if (k0 >= seen) continue;
    const int64_t base = (static_cast<int64_t>(page) * a.h_kv + hk) * bs * D + c * F;
    const T* kp = static_cast<const T*>(a.k) + base;
    const T* vp = static_cast<const T*>(a.v) + base;
    rot_u32x4 kr[U], vr[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = k0 + i * RPW + g;
      kr[i] = *reinterpret_cast<const rot_u32x4*>(kp + (r < seen ? r : seen - 1) * D);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int r = k0 + i * RPW + g;
      vr[i] = *reinterpret_cast<const rot_u32x4*>(vp + (r < seen ? r : seen - 1) * D);
      if (r >= seen) vr[i] = rot_u32x4{0, 0, 0, 0};  // hidden values add nothing, whatever they are
    }
    float s[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float t = 0.f;
      const T* ke = reinterpret_cast<const T*>(&kr[i]);
#pragma unroll
      for (int e = 0; e < F; ++e) t = fmaf(q[e], Elem<T>::load(ke, e), t);
      t = row_sum<LPR>(t);
      s[i] = k0 + i * RPW + g < seen ? t : -INFINITY;
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < U; ++i) top = fmaxf(top, s[i]);
    const float z = top > -INFINITY ? top : 0.f;
    const float old = __builtin_amdgcn_exp2f(m - z);
    l *= old;
#pragma unroll
    for (int e = 0; e < F; ++e) o[e] *= old;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float p = __builtin_amdgcn_exp2f(s[i] - z);
      l += p;
      const T* ve = reinterpret_cast<const T*>(&vr[i]);
#pragma unroll
      for (int e = 0; e < F; ++e) o[e] = fmaf(p, Elem<T>::load(ve, e), o[e]);
    }
    m = top;
  }
  // Lane groups, then waves.
#pragma unroll
  for (int off = LPR; off < 64; off <<= 1) {
    const float om = __shfl_xor(m, off), ol = __shfl_xor(l, off);
    const float top = fmaxf(m, om), z = top > -INFINITY ? top : 0.f;
    const float wa = __builtin_amdgcn_exp2f(m - z), wb = __builtin_amdgcn_exp2f(om - z);
    l = l * wa + ol * wb;
#pragma unroll
    for (int e = 0; e < F; ++e) o[e] = o[e] * wa + __shfl_xor(o[e], off) * wb;
    m = top;
  }
  if (g == 0) {
#pragma unroll
    for (int e = 0; e < F; ++e) s_o[wave][c * F + e] = o[e];
    if (c == 0) {
      s_m[wave] = m;
      s_l[wave] = l;
    }
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) top = fmaxf(top, s_m[w]);
  const float z = top > -INFINITY ? top : 0.f;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) total += s_l[w] * __builtin_amdgcn_exp2f(s_m[w] - z);
  for (int d = threadIdx.x; d < D; d += 64 * NW) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) x += s_o[w][d] * __builtin_amdgcn_exp2f(s_m[w] - z);
    if (a.splits == 1)
      Elem<T>::store(static_cast<T*>(a.out) + row * D, d, row_value(x, total));
    else
      a.part_o[(row * a.splits + blockIdx.y) * D + d] = x;
  }
  if (threadIdx.x == 0) {
    if (a.splits > 1) {
      a.part_ml[(row * a.splits + blockIdx.y) * 2] = top;
      a.part_ml[(row * a.splits + blockIdx.y) * 2 + 1] = total;
    } else if (a.lse) {
      a.lse[h * static_cast<int64_t>(a.p.tokens) + tok] = row_lse(top, total);
    }
  }
}

// Splits of a row merged: one wave per row.
template <typename T, int D>
__global__ void __launch_bounds__(64) merge_rows_kernel(RowArgs a) {
  const int64_t row = blockIdx.x;
  const int32_t tok = static_cast<int32_t>(row / a.h_q);
  if (locate(a.p, tok).pos < 0) return;
  const float* ml = a.part_ml + row * a.splits * 2;
  const float* po = a.part_o + row * a.splits * D;
  float top = -INFINITY;
  for (int i = 0; i < a.splits; ++i) top = fmaxf(top, ml[2 * i]);
  const float z = top > -INFINITY ? top : 0.f;
  float total = 0.f, o[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
  for (int i = 0; i < a.splits; ++i) {
    const float w = __builtin_amdgcn_exp2f(ml[2 * i] - z);
    total += ml[2 * i + 1] * w;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] += po[i * D + 64 * e + threadIdx.x] * w;
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    Elem<T>::store(static_cast<T*>(a.out) + row * D, 64 * e + threadIdx.x,
                   row_value(o[e], total));
  if (a.lse && threadIdx.x == 0)
    a.lse[(row % a.h_q) * static_cast<int64_t>(a.p.tokens) + tok] = row_lse(top, total);
}

// How a call is cut up, and its workspace.
struct PagedPlan {
  int64_t waves;   // per workgroup of attend_rows_kernel
  int64_t splits;  // parts of a query's chosen blocks
  size_t ml, o, ids, total;
};

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Keys per run of attend_rows_kernel.
int64_t run_keys(int64_t D, int dtype) { return 64 * 8 / (D / (dtype == MOBA_FP32 ? 4 : 8)); }

// Few queries: attend_rows_kernel chooses from the scores by itself.
bool chooses_itself(const moba_paged& c) { return scores_only(c) && !chunk_takes(c); }

PagedPlan plan_of(const moba_paged& c) {
  PagedPlan pl;
  const int64_t rows = c.tokens * c.h_q;
  const int64_t units = c.slots * cdiv(c.block_size, run_keys(c.head_dim, static_cast<int>(c.dtype)));
  // Few rows: wide workgroups, and several of them per row. With the choice of
  // the blocks, 32 heads of 128 over 32k keys: 256 rows by 16 waves 36 us, by 4
  // waves 39; 512 rows by 16 waves 68 us, by 4 waves 63, as two workgroups per
  // row (87 as one); 64 rows of 64k keys in 16 splits of 4 waves 25, in 4 of 16
  // waves 23.
  pl.waves = rows <= 256 && units > 4 ? 16 : 4;
  const int64_t splits = cdiv(1024, rows * pl.waves / 4);
  const int64_t most = cdiv(units, pl.waves);
  pl.splits = splits < most ? splits : most;
  const size_t parts = pl.splits > 1 ? static_cast<size_t>(rows * pl.splits) : 0;
  pl.ml = align256(sizeof(float) * 2 * parts);
  pl.o = align256(sizeof(float) * c.head_dim * parts);
  // The gate's scratch is free again when the blocks are chosen.
  const size_t gate = gate_workspace(c);
  if (chunk_takes(c)) {
    const size_t attend = chunk_plan(c).total;
    pl.total = attend > gate ? attend : gate;
  } else {
    pl.total = gate + pl.ml + pl.o;
  }
  // The chosen blocks, where the caller of moba_paged_attention has no use for them.
  pl.ids = chooses_itself(c) ? 0 : align256(sizeof(int32_t) * static_cast<size_t>(rows * c.slots));
  pl.total += pl.ids;
  return pl;
}

int check_attention(const moba_paged* c, Paged* p) {
  const int st = paged_of(c, p);
  if (st) return st;
  if (c->slots <= 0 || c->take < 0 || c->take + (c->always_current ? 1 : 0) > c->slots)
    return fail(MOBA_ERR_INVALID, "slots must hold the selected blocks");
  if (c->table_width > 65536) return fail(MOBA_ERR_UNSUPPORTED, "more than 65536 blocks per sequence");
  if (c->take > MOBA_PAGED_MAX_TAKE)
    return fail(MOBA_ERR_UNSUPPORTED, "more than " + std::to_string(MOBA_PAGED_MAX_TAKE) +
                                          " past blocks per query");
  if (c->tokens * c->h_q > ((int64_t(1) << 31) - 1) / c->slots)
    return fail(MOBA_ERR_UNSUPPORTED, "more than 2^31 - 1 (query, slot) entries");
  return MOBA_OK;
}

int check_workspace(const moba_paged* c, size_t need) {
  if (!c->workspace || static_cast<size_t>(c->workspace_bytes) < need)
    return fail(MOBA_ERR_WORKSPACE, "paged attention workspace too small");
  return MOBA_OK;
}

bool aligned(const void* p) { return p && on_16_bytes(p); }

}  // namespace

int paged_of(const moba_paged* c, Paged* p) {
  if (!c) return fail(MOBA_ERR_INVALID, "null pointer");
  constexpr int64_t kMax = (int64_t(1) << 31) - 1;
  for (int64_t n : {c->tokens, c->seqs, c->h_q, c->h_kv, c->head_dim, c->block_size,
                    c->table_width, c->n_pages}) {
    if (n <= 0) return fail(MOBA_ERR_INVALID, "non-positive shape argument");
    if (n > kMax) return fail(MOBA_ERR_UNSUPPORTED, "a size exceeds 2^31 - 1");
  }
  if (c->h_q % c->h_kv)
    return fail(MOBA_ERR_INVALID, "query heads " + std::to_string(c->h_q) +
                                      " not divisible by kv heads " + std::to_string(c->h_kv));
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(MOBA_ERR_UNSUPPORTED, "paged caches take head_dim 64, 128 or 256");
  if (c->block_size > 1024) return fail(MOBA_ERR_UNSUPPORTED, "block_size above 1024");
  if (c->dtype < 0 || c->dtype > MOBA_FP32)
    return fail(MOBA_ERR_UNSUPPORTED, "unknown dtype code");
  *p = Paged{c->block_table, c->seq_lens, c->cu_seqlens, static_cast<int32_t>(c->seqs),
             static_cast<int32_t>(c->table_width), static_cast<int32_t>(c->n_pages),
             static_cast<int32_t>(c->tokens), static_cast<int32_t>(c->even),
             static_cast<int32_t>(c->block_size)};
  if (!p->table || !p->seq_lens) return fail(MOBA_ERR_INVALID, "null pointer");
  if (!p->cu && (c->even <= 0 || c->even * c->seqs != c->tokens))
    return fail(MOBA_ERR_INVALID,
                "without cu_seqlens every sequence has the same number of new tokens");
  if (c->table_width * c->block_size > kMax)
    return fail(MOBA_ERR_UNSUPPORTED, "a sequence of the block table exceeds 2^31 - 1 tokens");
  return MOBA_OK;
}

}  // namespace moba

extern "C" int moba_paged_layout(moba_paged* c) {
  using namespace moba;
  Paged p;
  const int st = check_attention(c, &p);
  if (st) return st;
  c->workspace_bytes = static_cast<int64_t>(plan_of(*c).total);
  return MOBA_OK;
}

static int run_gate(const moba_paged* c, bool all_rows, void* stream) {
  using namespace moba;
  Paged p;
  int st = check_attention(c, &p);
  if (st) return st;
  if (!aligned(c->q) || !aligned(c->kbar) || !c->block_idx)
    return fail(MOBA_ERR_INVALID, "null or unaligned pointer");
  st = check_workspace(c, plan_of(*c).total);
  if (st) return st;
  return gate_run(*c, p, c->workspace, all_rows, as_stream(stream));
}

extern "C" int moba_paged_gate(const moba_paged* c, void* stream) { return run_gate(c, true, stream); }

// `keys`: scores to choose from, or null where c.block_idx holds the blocks.
static int run_attend(const moba_paged* c, const uint32_t* keys, void* stream) {
  using namespace moba;
  RowArgs a;
  int st = check_attention(c, &a.p);
  if (st) return st;
  if (!aligned(c->q) || !aligned(c->k) || !aligned(c->v) || !aligned(c->out) ||
      !(keys || c->block_idx))
    return fail(MOBA_ERR_INVALID, "null or unaligned pointer");
  const PagedPlan pl = plan_of(*c);
  st = check_workspace(c, pl.total);
  if (st) return st;
  hipStream_t s = as_stream(stream);
  if (chunk_takes(*c)) return chunk_attend(*c, a.p, c->workspace, s);
  char* scratch = static_cast<char*>(c->workspace) + gate_workspace(*c);
  a.q = c->q;
  a.k = c->k;
  a.v = c->v;
  a.block_idx = c->block_idx;
  a.keys = keys;
  a.out = c->out;
  a.lse = c->lse;
  a.part_ml = reinterpret_cast<float*>(scratch);
  a.part_o = reinterpret_cast<float*>(scratch + pl.ml);
  a.h_q = static_cast<int>(c->h_q);
  a.h_kv = static_cast<int>(c->h_kv);
  a.slots = static_cast<int>(c->slots);
  a.splits = static_cast<int>(pl.splits);
  a.take = static_cast<int>(c->take);
  a.current = c->always_current != 0;
  if (keys) a.slots = a.take + a.current;  // those it chooses; further ones are padding
  a.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(c->head_dim)));
  const int64_t rows = c->tokens * c->h_q;
  return MOBA_DISPATCH_DTYPE(static_cast<int>(c->dtype), T, [&] {
    auto go = [&](auto dim, auto nw, auto tm) {
      constexpr int D = decltype(dim)::value, NW = decltype(nw)::value, TM = decltype(tm)::value;
      // A launch holds fewer than 2^32 threads (per axis).
      constexpr int64_t most = (int64_t(1) << 32) / (64 * NW) - 1;
      int rc = MOBA_OK;
      for (a.row0 = 0; a.row0 < rows && !rc; a.row0 += most) {
        const int64_t n = rows - a.row0 < most ? rows - a.row0 : most;
        hipLaunchKernelGGL((attend_rows_kernel<T, D, NW, TM>),
                           dim3(static_cast<unsigned>(n), static_cast<unsigned>(a.splits)),
                           dim3(64 * NW), 0, s, a);
        rc = check_launch("moba_paged_attend");
      }
      if (rc || a.splits == 1) return rc;  // splits: of at most a few thousand rows
      hipLaunchKernelGGL((merge_rows_kernel<T, D>), dim3(static_cast<unsigned>(rows)), dim3(64), 0, s, a);
      return check_launch("moba_paged_attend (merge)");
    };
    auto lists = [&](auto dim, auto nw) {
      if (!keys) return go(dim, nw, std::integral_constant<int, 0>{});
      if (a.take <= 8) return go(dim, nw, std::integral_constant<int, 8>{});
      if (a.take <= 16) return go(dim, nw, std::integral_constant<int, 16>{});
      return go(dim, nw, std::integral_constant<int, 32>{});
    };
    auto waves = [&](auto dim) {
      if (pl.waves == 4) return lists(dim, std::integral_constant<int, 4>{});
      return lists(dim, std::integral_constant<int, 16>{});
    };
    switch (c->head_dim) {
      case 64: return waves(std::integral_constant<int, 64>{});
      case 128: return waves(std::integral_constant<int, 128>{});
      default: return waves(std::integral_constant<int, 256>{});
    }
  });
}

extern "C" int moba_paged_attend(const moba_paged* c, void* stream) { return run_attend(c, nullptr, stream); }

extern "C" int moba_paged_attention(const moba_paged* c, void* stream) {
  using namespace moba;
  Paged p;
  int st = check_attention(c, &p);
  if (st) return st;
  const PagedPlan pl = plan_of(*c);
  if (chooses_itself(*c)) {
    if (!aligned(c->q) || !aligned(c->kbar)) return fail(MOBA_ERR_INVALID, "null or unaligned pointer");
    st = check_workspace(c, pl.total);
    if (!st) st = gate_scores(*c, p, c->workspace, as_stream(stream));
    return st ? st : run_attend(c, static_cast<const uint32_t*>(c->workspace), stream);
  }
  moba_paged call = *c;
  if (!call.block_idx && call.workspace)
    call.block_idx = reinterpret_cast<int32_t*>(static_cast<char*>(call.workspace) + pl.total - pl.ids);
  st = run_gate(&call, false, stream);
  return st ? st : run_attend(&call, nullptr, stream);
}
