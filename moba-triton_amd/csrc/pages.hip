// Pages of a cache: new tokens appended (normed and rotated on the way), and
// pages copied.
#include "paged.h"
#include "rotary.h"

namespace moba {

namespace {

struct AppendArgs {
  Paged p;
  const void *q, *k, *v;   // [tokens, heads, D] by strides (elements)
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void* q_out;             // [tokens, h_q, D]
  void *k_pages, *v_pages, *kbar;
  const void *wq, *wk;     // [D] or null
  const float *cosv, *sinv;
  int64_t table_len;
  int h_q, h_kv, rotary, w_f32;
  float eps;
};

// The piece-th run of new tokens that share a page: sequence, its first
// position and its end. Sequences are counted 64 at a time by a wave's lanes.
struct Piece {
  int32_t seq, begin, end;  // positions; seq -1: no such piece
  int32_t tok;              // token of `begin`
};

__device__ inline Piece find_piece(const Paged& p, int32_t piece) {
  const int lane = threadIdx.x & 63;
  int32_t before = 0, reach = 0;
  for (int32_t base = 0; base < p.seqs; base += 64) {
    const NewTokens r = counted_tokens(p, base, reach);
    const int32_t lo = r.len - r.n;
    const int32_t mine = r.n ? (r.len - 1) / p.block - lo / p.block + 1 : 0;
    int32_t upto = mine;  // inclusive sum over the lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t y = __shfl_up(upto, off);
      if (lane >= off) upto += y;
    }
    const uint64_t past = __ballot(before + upto > piece);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int32_t skip = piece - before - (__shfl(upto, l) - __shfl(mine, l));
      const int32_t from = __shfl(lo, l), len = __shfl(r.len, l), first = __shfl(r.first, l);
      Piece out;
      out.seq = base + l;
      const int64_t edge = (static_cast<int64_t>(from / p.block) + skip) * p.block;
      out.begin = skip ? static_cast<int32_t>(edge) : from;
      out.end = edge + p.block < len ? static_cast<int32_t>(edge + p.block) : len;
      out.tok = first + (out.begin - from);
      return out;
    }
    before += __shfl(upto, 63);
  }
  return Piece{-1, 0, 0, 0};
}

// Memory-bound on prompts (5 of 1000 to 4096 tokens, 16 + 4 heads of 128 in
// bf16: 33 us, 26 at the rate of a large copy); on single tokens of 64 sequences
// 12 us, most of it the chain lengths -> table -> page -> keys of a block that
// the token completes.
//
// One workgroup per run of new tokens on one page and (y) kv head, or four
// query heads: y < h_kv writes K and V rows into the page and, where the run
// fills the page's last row, the block's representative; the others write
// rows of q_out. Rows go through registers once.
//
// kbar is pool.hip's: the exact sum (float64; for 16-bit types it does not
// depend on the order) rounded to float32 and to the type, the quotient
// rounded to the type. Keys written before are read back from the page.
constexpr int kAppendThreads = 256;
constexpr int kQHeads = 4;

template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(AppendArgs a) {
  constexpr int D = 16 * LPR;
  constexpr int G = kAppendThreads / LPR;  // lane groups: rows at a time
  __shared__ double sums[kAppendThreads / 64][D];
  const Piece pc = find_piece(a.p, blockIdx.x);
  if (pc.seq < 0) return;
  const int lane = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const RotLane rl = rot_lane(lane, a.rotary, IL);
  const int n = pc.end - pc.begin;
  if (static_cast<int>(blockIdx.y) >= a.h_kv) {  // queries
    const int h0 = (static_cast<int>(blockIdx.y) - a.h_kv) * kQHeads;
    const int heads = a.h_q - h0 < kQHeads ? a.h_q - h0 : kQHeads;
    float w[16];
    if (a.wq) load16<T>(a.wq, a.w_f32, rl, w);
    constexpr int R = 4;
    for (int i0 = g; i0 < n * heads; i0 += R * G) {
      RawRow<T> raw[R];
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const int i = min(i0 + u * G, n * heads - 1);
        raw[u].load(static_cast<const T*>(a.q) + static_cast<int64_t>(pc.tok + i / heads) * a.q_tok +
                        (h0 + i % heads) * a.q_head, rl);
      }
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const int last = n * heads - 1, i = min(i0 + u * G, last);
        const int t = i / heads, h = h0 + i % heads;
        float c[8], sn[8];
        rot_turn(rl, a.cosv, a.sinv, a.rotary, pc.begin + t, a.table_len, c, sn);
        float v[16];
        raw[u].widen(v);
        if (a.wq) {
          const float r = rsqrtf(row_sum<LPR>(square_sum(v)) * (1.f / D) + a.eps);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
        }
        rotate16<IL>(rl, c, sn, v);
        raw[u].narrow(v);
        if (i0 + u * G <= last)
          raw[u].store(static_cast<T*>(a.q_out) + (static_cast<int64_t>(pc.tok + t) * a.h_q + h) * D, rl);
      }
    }
    return;
  }
  const int h = blockIdx.y;
  const int bs = a.p.block;
  const int32_t blk = pc.begin / bs;
  const int32_t page = page_of(a.p, pc.seq, blk);
  if (page < 0) return;  // no page: the tokens have no place
  const int first = pc.begin - blk * bs;  // first new row of the page
  const bool full = first + n == bs;
  const int64_t base = (static_cast<int64_t>(page) * a.h_kv + h) * bs * D;
  T* kp = static_cast<T*>(a.k_pages) + base;
  T* vp = static_cast<T*>(a.v_pages) + base;
  float w[16];
  if (a.wk) load16<T>(a.wk, a.w_f32, rl, w);
  double sum[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.0;
  if (full) {
    constexpr int R = 4;
    for (int i0 = g; i0 < first; i0 += R * G) {
      RawRow<T> raw[R];
#pragma unroll
      for (int u = 0; u < R; ++u) raw[u].load(kp + static_cast<int64_t>(min(i0 + u * G, first - 1)) * D, rl);
#pragma unroll
      for (int u = 0; u < R; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          sum[e] += i0 + u * G < first ? static_cast<double>(raw[u].element(e)) : 0.0;
    }
  }
  constexpr int R = 2;
  for (int i0 = g; i0 < n; i0 += R * G) {
    RawRow<T> raw[R], rv[R];
    float c[R][8], sn[R][8];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int i = min(i0 + u * G, n - 1);
      const int64_t tok = pc.tok + i;
      raw[u].load(static_cast<const T*>(a.k) + tok * a.k_tok + h * a.k_head, rl);
      rv[u].load(static_cast<const T*>(a.v) + tok * a.v_tok + h * a.v_head, rl);
      rot_turn(rl, a.cosv, a.sinv, a.rotary, pc.begin + i, a.table_len, c[u], sn[u]);
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int i = i0 + u * G;
      float v[16];
      raw[u].widen(v);
      if (a.wk) {
        const float r = rsqrtf(row_sum<LPR>(square_sum(v)) * (1.f / D) + a.eps);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
      }
      rotate16<IL>(rl, c[u], sn[u], v);
      raw[u].narrow(v);
      if (i < n) {
        raw[u].store(kp + static_cast<int64_t>(first + i) * D, rl);
        rv[u].store(vp + static_cast<int64_t>(first + i) * D, rl);
        if (full) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sum[e] += static_cast<double>(raw[u].element(e));
        }
      }
    }
  }
  if (!full) return;  // the same in the whole workgroup
#pragma unroll
  for (int e = 0; e < 16; ++e)
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1) sum[e] += __shfl_xor(sum[e], off);
  if ((threadIdx.x & 63) < LPR) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sums[threadIdx.x >> 6][rl.lo + e] = sum[e];
      sums[threadIdx.x >> 6][rl.hi + e] = sum[8 + e];
    }
  }
  __syncthreads();
  T* dst = static_cast<T*>(a.kbar) + (static_cast<int64_t>(page) * a.h_kv + h) * D;
  for (int d = threadIdx.x; d < D; d += kAppendThreads) {
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < kAppendThreads / 64; ++i) t += sums[i][d];
    Elem<T>::store(dst, d, Elem<T>::round(static_cast<float>(t)) / static_cast<float>(bs));
  }
}

// Up to this many (source, destination) pairs travel in the kernel's
// arguments: a host list needs no copy to the device, also under capture.
constexpr int kHostPairs = 256;
struct CopyPairs {
  int32_t src[kHostPairs], dst[kHostPairs];
};
struct CopyArgs {
  uint4* buf[3];           // K, V, kbar: [layers, pages, bytes]
  int64_t page16[3];       // 16-byte pieces of a page
  int64_t pages;
  const int32_t* src;      // device lists, or null: the pairs below
  const int32_t* dst;
  int64_t first;           // first pair of this launch
};

// grid (pieces of a page's K, V and kbar, pairs, layers); a workgroup moves
// kCopy pieces per thread, all in flight. Memory-bound: 180 pages of 16 layers (8
// heads, blocks of 128 x 128 in bf16, 3.0 GB) in 600 us, 5.1 TB/s; 8 pages in 27.
constexpr int kCopy = 4;
__global__ void __launch_bounds__(256) copy_kernel(CopyArgs a, CopyPairs list) {
  const int64_t pair = blockIdx.y;
  const int32_t src = a.src ? a.src[a.first + pair] : list.src[pair];
  const int32_t dst = a.dst ? a.dst[a.first + pair] : list.dst[pair];
  if (src < 0 || dst < 0 || src >= a.pages || dst >= a.pages) return;
  // Which buffer this workgroup's run belongs to.
  int64_t x = blockIdx.x;
  int b = 0;
  for (; b < 2; ++b) {
    const int64_t runs = (a.page16[b] + 256 * kCopy - 1) / (256 * kCopy);
    if (x < runs) break;
    x -= runs;
  }
  const int64_t n = a.page16[b];
  const uint4* from = a.buf[b] + (blockIdx.z * a.pages + src) * n;
  uint4* to = a.buf[b] + (blockIdx.z * a.pages + dst) * n;
  const int64_t i0 = x * 256 * kCopy + threadIdx.x;
  uint4 r[kCopy];
#pragma unroll
  for (int u = 0; u < kCopy; ++u)
    if (i0 + 256 * u < n) r[u] = from[i0 + 256 * u];
#pragma unroll
  for (int u = 0; u < kCopy; ++u)
    if (i0 + 256 * u < n) to[i0 + 256 * u] = r[u];
}

}  // namespace

}  // namespace moba

extern "C" int moba_append_tokens(const moba_paged* c, const void* k_new, const void* v_new,
                                  const int64_t* strides, void* q_out, const float* cos_table,
                                  const float* sin_table, const void* q_weight,
                                  const void* k_weight, int64_t rotary, int64_t table_len,
                                  int interleaved, double eps, int weight_dtype, void* stream) {
  using namespace moba;
  AppendArgs a;
  int st = paged_of(c, &a.p);
  if (!st) st = check_rotary(c->head_dim, rotary, table_len, cos_table, sin_table,
                             static_cast<int>(c->dtype), weight_dtype);
  if (st) return st;
  if (!c->q || !k_new || !v_new || !strides || !q_out || !c->k || !c->v || !c->kbar)
    return fail(MOBA_ERR_INVALID, "null pointer");
  for (const void* p : {c->q, k_new, v_new, static_cast<const void*>(q_out),
                        static_cast<const void*>(c->k), static_cast<const void*>(c->v),
                        static_cast<const void*>(c->kbar)})
    if (!on_16_bytes(p)) return fail(MOBA_ERR_INVALID, "rows must start on 16-byte boundaries");
  for (int i = 0; i < 6; ++i)
    if (strides[i] % (c->dtype == MOBA_FP32 ? 4 : 8))
      return fail(MOBA_ERR_INVALID, "strides must be multiples of 16 bytes");
  a.q = c->q;
  a.k = k_new;
  a.v = v_new;
  a.q_tok = strides[0]; a.q_head = strides[1];
  a.k_tok = strides[2]; a.k_head = strides[3];
  a.v_tok = strides[4]; a.v_head = strides[5];
  a.q_out = q_out;
  a.k_pages = c->k;
  a.v_pages = c->v;
  a.kbar = c->kbar;
  a.wq = q_weight;
  a.wk = k_weight;
  a.cosv = cos_table;
  a.sinv = sin_table;
  a.table_len = table_len;
  a.h_q = static_cast<int>(c->h_q);
  a.h_kv = static_cast<int>(c->h_kv);
  a.rotary = static_cast<int>(rotary);
  a.w_f32 = weight_dtype == MOBA_FP32;
  a.eps = static_cast<float>(eps);
  // Runs of new tokens on one page: a sequence of n tokens has at most
  // (n - 1) / block + 2, and never more than n.
  const int64_t runs = cdiv(a.p.tokens, a.p.block) + 2 * static_cast<int64_t>(a.p.seqs);
  dim3 grid(static_cast<unsigned>(runs < a.p.tokens ? runs : a.p.tokens),
            static_cast<unsigned>(a.h_kv + cdiv(a.h_q, kQHeads)));
  if (grid.y > 65535) return fail(MOBA_ERR_UNSUPPORTED, "append: too many heads");
  if (grid.x >= 1u << 24)  // of 256 threads: a launch holds fewer than 2^32
    return fail(MOBA_ERR_UNSUPPORTED, "append: too many tokens");
  return MOBA_DISPATCH_DTYPE(static_cast<int>(c->dtype), T, [&] {
    auto run = [&](auto lpr, auto il) {
      hipLaunchKernelGGL((append_kernel<T, decltype(lpr)::value, decltype(il)::value>), grid, dim3(kAppendThreads), 0,
                         as_stream(stream), a);
      return check_launch("moba_append_tokens");
    };
    auto go = [&](auto lpr) {
      return interleaved ? run(lpr, std::true_type{}) : run(lpr, std::false_type{});
    };
    switch (c->head_dim) {
      case 64: return go(std::integral_constant<int, 4>{});
      case 128: return go(std::integral_constant<int, 8>{});
      default: return go(std::integral_constant<int, 16>{});
    }
  });
}

extern "C" int moba_copy_pages(void* k, void* v, void* kbar, const int32_t* src,
                               const int32_t* dst, int64_t n, int on_host, int64_t layers,
                               int64_t pages, int64_t h_kv, int64_t block_size, int64_t head_dim,
                               int dtype, void* stream) {
  using namespace moba;
  if (n < 0 || layers <= 0 || pages <= 0 || h_kv <= 0 || block_size <= 0 || head_dim <= 0)
    return fail(MOBA_ERR_INVALID, "non-positive shape argument");
  if (n == 0) return MOBA_OK;
  if (!k || !v || !kbar || !src || !dst) return fail(MOBA_ERR_INVALID, "null pointer");
  if (dtype < 0 || dtype > MOBA_FP32) return fail(MOBA_ERR_UNSUPPORTED, "unknown dtype code");
  const int64_t row = h_kv * head_dim * (dtype == MOBA_FP32 ? 4 : 2);
  if (row % 16 || !on_16_bytes(k) || !on_16_bytes(v) || !on_16_bytes(kbar))
    return fail(MOBA_ERR_INVALID, "pages must lie on 16-byte boundaries");
  if (layers > 65535 || pages > (int64_t(1) << 31) - 1)
    return fail(MOBA_ERR_UNSUPPORTED, "copy_pages: too many layers or pages");
  CopyArgs a;
  a.buf[0] = static_cast<uint4*>(k);
  a.buf[1] = static_cast<uint4*>(v);
  a.buf[2] = static_cast<uint4*>(kbar);
  a.page16[0] = a.page16[1] = row / 16 * block_size;
  a.page16[2] = row / 16;
  a.pages = pages;
  a.src = on_host ? nullptr : src;
  a.dst = on_host ? nullptr : dst;
  int64_t runs = 0;
  for (int64_t p : a.page16) runs += cdiv(p, 256 * kCopy);
  if (runs > (int64_t(1) << 31) - 1) return fail(MOBA_ERR_UNSUPPORTED, "copy_pages: page too large");
  CopyPairs list;
  const int64_t most = on_host ? kHostPairs : 65535;
  for (a.first = 0; a.first < n; a.first += most) {
    const int64_t m = n - a.first < most ? n - a.first : most;
    for (int64_t i = 0; on_host && i < m; ++i) {
      list.src[i] = src[a.first + i];
      list.dst[i] = dst[a.first + i];
    }
    hipLaunchKernelGGL(copy_kernel, dim3(static_cast<unsigned>(runs), static_cast<unsigned>(m),
                                         static_cast<unsigned>(layers)),
                       dim3(256), 0, as_stream(stream), a, list);
    const int st = check_launch("moba_copy_pages");
    if (st) return st;
  }
  return MOBA_OK;
}
