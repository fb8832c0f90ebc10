// Norm of queries and keys per head with the position rotation in the same
// pass, forward and backward.
//
//   r = (mean_d x_d^2 + eps)^-1/2,  n = x r w
//   y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin   for the feature pairs
//   (a, b) of the first `rotary` features (halves: b = a + rotary / 2;
//   neighbours: a = 2i, b = 2i + 1), y = n beyond them.
//
// All in float32, rounded once to the type. Backward, with g = R^T dy, the
// normalised row x r and h = g w:
//
//   dx = r (h - (x r) mean(h (x r))),  dw = sum over rows of g (x r).
//
// A row (one head of one token) belongs to D / 16 adjacent lanes, 16 features
// each in two 16-byte pieces (four in float32) that hold both members of
// their pairs, so the rotation crosses no lanes and the row sums take
// log2(D / 16) shuffles. A lane group walks heads of one token with that
// token's cosines and sines in registers, kRows rows in flight.
//
// dw: every workgroup sums its rows in float32 (20 rows per lane in the call
// below, 320 at 524288 tokens, each off by at most 2^-24 of the sum of the terms'
// magnitudes), its lanes meet in LDS in a fixed order, and a second kernel adds
// the workgroups' sums in float64 in order: the result depends on the shape only.
//
// Memory-bound: 32768 tokens of 32 + 8 heads of 128 in bf16 take 131 us forward
// (671 MB, 5.1 TB/s; a large device copy reaches 4.9 here) and 211 + 7 backward
// (1.0 GB, 4.8 TB/s). Rows in flight as an array that the compiler cannot keep
// in registers (a loop left early, the pairing chosen at run time) took 334 and
// 449. 8 tokens of 16 + 4 heads: 5 us, a launch and three dependent loads.
#include "rotary.h"

#include <initializer_list>

namespace moba {

namespace {

// One tensor of a call: x [batch, seq, heads, D] by strides (elements),
// y (forward: the result; backward: dx) and dy contiguous.
struct RotSide {
  const void* x;
  const void* dy;
  void* y;
  const void* w;      // [D], or null: no norm
  int64_t sb, ss, sh; // strides of x
  int heads;
  int slices_log2;    // 2^ lane groups share a token's heads
  float* partial;     // backward: dw sums [workgroups, D]
  int blocks;         // workgroups of this side
  int flat;           // the batch axis continues the token axis: sb = seq * ss
};

struct RotArgs {
  RotSide side[2];  // queries, keys
  const float* cosv;
  const float* sinv;
  const int32_t* positions;  // [batch * seq], or null: 0, 1, .. in each row
  uint32_t tokens, seq;
  int64_t table_len;
  int rotary, w_f32;
  float eps;
};

// Workgroups' sizes and the rows a lane group holds at a time.
constexpr int kThreads = 256;
constexpr int kRows = 4;

// Element offset of token `tok`'s first head.
__device__ inline int64_t token_offset(const RotArgs& a, const RotSide& s, uint32_t tok) {
  if (s.flat) return tok * s.ss;
  const uint32_t b = tok / a.seq;
  return b * s.sb + (tok - b * a.seq) * s.ss;
}

__device__ inline int32_t position_of(const RotArgs& a, uint32_t tok) {
  if (a.positions) return a.positions[tok];
  return static_cast<int32_t>(tok % a.seq);
}

// Workgroups stride over the side's lane groups' work, (token, slice of its
// heads) pairs: one reading of the weights serves many rows.
template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kThreads) norm_rotate_kernel(RotArgs a) {
  constexpr int D = 16 * LPR;
  constexpr uint32_t kGroups = kThreads / LPR;
  const bool second = static_cast<int>(blockIdx.x) >= a.side[0].blocks;
  const RotSide s = a.side[second];
  const uint32_t block = blockIdx.x - (second ? a.side[0].blocks : 0);
  const int lane = threadIdx.x % LPR;
  const RotLane rl = rot_lane(lane, a.rotary, IL);
  float w[16];
  if (s.w) load16<T>(s.w, a.w_f32, rl, w);
  const int slices = 1 << s.slices_log2;
  const uint64_t work = static_cast<uint64_t>(a.tokens) << s.slices_log2;
  for (uint64_t group = static_cast<uint64_t>(block) * kGroups + threadIdx.x / LPR; group < work;
       group += static_cast<uint64_t>(s.blocks) * kGroups) {
    const uint32_t tok = static_cast<uint32_t>(group >> s.slices_log2);
    const int slice = static_cast<int>(group & (slices - 1));
    if (slice >= s.heads) continue;
    const T* x = static_cast<const T*>(s.x) + token_offset(a, s, tok);
    T* y = static_cast<T*>(s.y) + static_cast<int64_t>(tok) * s.heads * D;
    float c[8], sn[8];
    rot_turn(rl, a.cosv, a.sinv, a.rotary, position_of(a, tok), a.table_len, c, sn);
    for (int h0 = slice; h0 < s.heads; h0 += kRows << s.slices_log2) {
      RawRow<T> raw[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int h = h0 + (i << s.slices_log2);
        raw[i].load(x + (h < s.heads ? h : h0) * s.sh, rl);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int h = h0 + (i << s.slices_log2);
        float v[16];
        raw[i].widen(v);
        if (s.w) {
          const float r = rsqrtf(row_sum<LPR>(square_sum(v)) * (1.f / D) + a.eps);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
        }
        rotate16<IL>(rl, c, sn, v);
        raw[i].narrow(v);
        if (h < s.heads) raw[i].store(y + h * D, rl);
      }
    }
  }
}

// dx, and this workgroup's share of dw. Workgroups of a side stride over its
// lane groups' work, so the number of partial sums is bounded.
template <typename T, int LPR, bool IL>
__global__ void __launch_bounds__(kThreads) norm_rotate_bwd_kernel(RotArgs a) {
  constexpr int D = 16 * LPR;
  constexpr int kGroups = kThreads / LPR;  // lane groups of the workgroup
  constexpr int R = 2;                     // rows in flight: x and dy of each
  __shared__ float sums[kThreads / 64][D];
  const bool second = static_cast<int>(blockIdx.x) >= a.side[0].blocks;
  const RotSide s = a.side[second];
  const int64_t block = static_cast<int64_t>(blockIdx.x) - (second ? a.side[0].blocks : 0);
  const int lane = threadIdx.x % LPR;
  const RotLane rl = rot_lane(lane, a.rotary, IL);
  float w[16], dw[16];
  if (s.w) load16<T>(s.w, a.w_f32, rl, w);
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[e] = 0.f;
  const int slices = 1 << s.slices_log2;
  const uint64_t work = static_cast<uint64_t>(a.tokens) << s.slices_log2;
  for (uint64_t group = static_cast<uint64_t>(block) * kGroups + threadIdx.x / LPR; group < work;
       group += static_cast<uint64_t>(s.blocks) * kGroups) {
    const uint32_t tok = static_cast<uint32_t>(group >> s.slices_log2);
    const int slice = static_cast<int>(group & (slices - 1));
    if (slice >= s.heads) continue;
    const T* x = static_cast<const T*>(s.x) + token_offset(a, s, tok);
    const T* dy = static_cast<const T*>(s.dy) + static_cast<int64_t>(tok) * s.heads * D;
    T* dx = static_cast<T*>(s.y) + static_cast<int64_t>(tok) * s.heads * D;
    float c[8], sn[8];
    rot_turn(rl, a.cosv, a.sinv, a.rotary, position_of(a, tok), a.table_len, c, sn);
    for (int h0 = slice; h0 < s.heads; h0 += R << s.slices_log2) {
      RawRow<T> rx[R], rg[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int hi = h0 + (i << s.slices_log2);
        const int h = hi < s.heads ? hi : h0;
        rg[i].load(dy + h * D, rl);
        if (s.w) rx[i].load(x + h * s.sh, rl);
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int h = h0 + (i << s.slices_log2);
        const bool in = h < s.heads;  // a row past the last counts nowhere
        float g[16];
        rg[i].widen(g);
        unrotate16<IL>(rl, c, sn, g);
        if (s.w) {
          float v[16];
          rx[i].widen(v);
          const float r = rsqrtf(row_sum<LPR>(square_sum(v)) * (1.f / D) + a.eps);
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            v[e] *= r;
            dw[e] = in ? fmaf(g[e], v[e], dw[e]) : dw[e];
            g[e] *= w[e];
            dot = fmaf(g[e], v[e], dot);
          }
          dot = row_sum<LPR>(dot) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 16; ++e) g[e] = r * (g[e] - v[e] * dot);
        }
        rg[i].narrow(g);
        if (in) rg[i].store(dx + h * D, rl);
      }
    }
  }
  if (!s.w) return;  // the side's whole workgroup
  // Lane groups of a wave by shuffles, waves through LDS.
#pragma unroll
  for (int e = 0; e < 16; ++e)
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1) dw[e] += __shfl_xor(dw[e], off);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < LPR) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sums[wave][rl.lo + e] = dw[e];
      sums[wave][rl.hi + e] = dw[8 + e];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < kThreads / 64; ++v) t += sums[v][d];
    s.partial[block * D + d] = t;
  }
}

// dw[d] = sum over the workgroups' partial sums, float64, in a fixed order:
// 64 threads per feature take every 64th workgroup and meet in LDS (16
// threads per feature: 15 us for 1638 workgroups of 128 features, 64: 7).
// grid (D / 16, 2).
template <typename W>
__global__ void __launch_bounds__(1024)
norm_weight_kernel(const float* __restrict__ pq, int nq, W* __restrict__ dwq,
                   const float* __restrict__ pk, int nk, W* __restrict__ dwk, int D) {
  const float* p = blockIdx.y ? pk : pq;
  const int n = blockIdx.y ? nk : nq;
  W* out = blockIdx.y ? dwk : dwq;
  if (!out) return;
  // Lanes along the features: 64-byte reads.
  __shared__ double part[64][17];
  const int d = threadIdx.x & 15, j = threadIdx.x >> 4;
  const int feature = blockIdx.x * 16 + d;
  double t = 0.0;
#pragma unroll 8
  for (int i = j; i < n; i += 64) t += static_cast<double>(p[static_cast<int64_t>(i) * D + feature]);
  part[j][d] = t;
  __syncthreads();
  if (j >= 4) return;
  for (int i = j + 4; i < 64; i += 4) t += part[i][d];
  t += __shfl_xor(t, 16);
  t += __shfl_xor(t, 32);
  if (j == 0) Elem<W>::store(out, feature, static_cast<float>(t));
}

int check(int64_t batch, int64_t seq, int64_t h_q, int64_t h_kv, int64_t D, int64_t rotary,
          int64_t table_len, const void* cosv, const void* sinv, int dtype, int w_dtype) {
  if (batch <= 0 || seq <= 0 || h_q <= 0 || h_kv <= 0)
    return fail(MOBA_ERR_INVALID, "non-positive shape argument");
  const int st = check_rotary(D, rotary, table_len, cosv, sinv, dtype, w_dtype);
  if (st) return st;
  if (batch > INT32_MAX / seq)
    return fail(MOBA_ERR_UNSUPPORTED, "norm_rotate: more than 2^31 - 1 tokens");
  if (h_q > 65536 || h_kv > 65536) return fail(MOBA_ERR_UNSUPPORTED, "norm_rotate: too many heads");
  return MOBA_OK;
}

// Rows move in 16-byte pieces.
int check_rows(std::initializer_list<const void*> rows, const int64_t* strides, int dtype) {
  for (const void* p : rows) {
    if (!p) return fail(MOBA_ERR_INVALID, "null pointer");
    if (!on_16_bytes(p)) return fail(MOBA_ERR_INVALID, "rows must start on 16-byte boundaries");
  }
  if (!strides) return fail(MOBA_ERR_INVALID, "null pointer");
  for (int i = 0; i < 6; ++i)
    if (strides[i] % (dtype == MOBA_FP32 ? 4 : 8))
      return fail(MOBA_ERR_INVALID, "strides must be multiples of 16 bytes");
  return MOBA_OK;
}

// log2 of the lane groups per token: a group holds kRows heads at a time. (A
// group for each head takes longer at every length, 32 + 8 heads of 128 in
// bf16: 64 tokens 5.0 us for 4.9, 1024 tokens 10.6 for 7.4, 4096 25.4 for 17.9.)
int slices_log2(int64_t heads) {
  const int64_t want = heads / kRows;
  int n = 0;
  while ((int64_t(2) << n) <= want) ++n;
  return n;
}

template <typename F>
int with_lanes(int64_t D, int interleaved, F&& go) {
  auto pairs = [&](auto lpr) {
    return interleaved ? go(lpr, std::true_type{}) : go(lpr, std::false_type{});
  };
  switch (D) {
    case 32: return pairs(std::integral_constant<int, 2>{});
    case 64: return pairs(std::integral_constant<int, 4>{});
    case 128: return pairs(std::integral_constant<int, 8>{});
    case 256: return pairs(std::integral_constant<int, 16>{});
    case 512: return pairs(std::integral_constant<int, 32>{});
    default: return pairs(std::integral_constant<int, 64>{});
  }
}

// Workgroups of a call, at most kMaxBlocks, shared by the sides' rows.
constexpr int64_t kMaxBlocks = 2048;
void set_blocks(RotArgs* a, int64_t head_dim) {
  const int64_t h_q = a->side[0].heads, h_kv = a->side[1].heads;
  int64_t share = kMaxBlocks * h_q / (h_q + h_kv);
  share = share < 1 ? 1 : (share < kMaxBlocks ? share : kMaxBlocks - 1);
  for (int i = 0; i < 2; ++i) {
    RotSide& s = a->side[i];
    const int64_t need = cdiv(static_cast<int64_t>(a->tokens) << s.slices_log2, kThreads / (head_dim / 16));
    const int64_t most = i ? kMaxBlocks - share : share;
    s.blocks = static_cast<int>(need < most ? need : most);
  }
}

RotArgs make_args(const void* q, const void* k, void* yq, void* yk, const float* cosv,
                  const float* sinv, const int32_t* positions, const void* wq, const void* wk,
                  int64_t batch, int64_t seq, int64_t h_q, int64_t h_kv, const int64_t* strides,
                  int64_t rotary, int64_t table_len, double eps, int w_dtype) {
  RotArgs a;
  const void* x[2] = {q, k};
  void* y[2] = {yq, yk};
  const void* w[2] = {wq, wk};
  const int64_t heads[2] = {h_q, h_kv};
  for (int i = 0; i < 2; ++i) {
    RotSide& s = a.side[i];
    s = RotSide{x[i], nullptr, y[i], w[i], strides[3 * i], strides[3 * i + 1], strides[3 * i + 2],
                static_cast<int>(heads[i]), slices_log2(heads[i]), nullptr, 0, 0};
    s.flat = batch == 1 || s.sb == seq * s.ss;
  }
  a.cosv = cosv;
  a.sinv = sinv;
  a.positions = positions;
  a.tokens = static_cast<uint32_t>(batch * seq);
  a.seq = static_cast<uint32_t>(seq);
  a.table_len = table_len;
  a.rotary = static_cast<int>(rotary);
  a.w_f32 = w_dtype == MOBA_FP32;
  a.eps = static_cast<float>(eps);
  return a;
}

}  // namespace

int check_rotary(int64_t D, int64_t rotary, int64_t table_len, const void* cosv, const void* sinv,
                 int dtype, int w_dtype) {
  if (D < 32 || D > 1024 || (D & (D - 1)))
    return fail(MOBA_ERR_UNSUPPORTED, "head_dim must be a power of two from 32 to 1024");
  if (rotary < 0 || rotary > D || rotary % 16)
    return fail(MOBA_ERR_INVALID, "rotated features must be a multiple of 16 of at most head_dim");
  if (rotary && (!cosv || !sinv || table_len <= 0))
    return fail(MOBA_ERR_INVALID, "rotation without cos / sin tables");
  if (rotary && !(on_16_bytes(cosv) && on_16_bytes(sinv)))
    return fail(MOBA_ERR_INVALID, "cos / sin tables must start on 16-byte boundaries");
  if (w_dtype != MOBA_FP32 && w_dtype != dtype)
    return fail(MOBA_ERR_INVALID, "norm weights must be float32 or of the input type");
  return MOBA_OK;
}

}  // namespace moba

extern "C" int moba_norm_rotate(const void* q, const void* k, void* q_out, void* k_out,
                                const float* cos_table, const float* sin_table,
                                const int32_t* positions, const void* q_weight,
                                const void* k_weight, int64_t batch, int64_t seq_len, int64_t h_q,
                                int64_t h_kv, int64_t head_dim, const int64_t* strides,
                                int64_t rotary, int64_t table_len, int interleaved, double eps,
                                int dtype, int weight_dtype, void* stream) {
  using namespace moba;
  int st = check(batch, seq_len, h_q, h_kv, head_dim, rotary, table_len, cos_table, sin_table,
                 dtype, weight_dtype);
  if (!st) st = check_rows({q, k, q_out, k_out}, strides, dtype);
  if (st) return st;
  RotArgs a = make_args(q, k, q_out, k_out, cos_table, sin_table, positions, q_weight, k_weight,
                        batch, seq_len, h_q, h_kv, strides, rotary, table_len, eps,
                        weight_dtype);
  set_blocks(&a, head_dim);
  return MOBA_DISPATCH_DTYPE(dtype, T, [&] {
    return with_lanes(head_dim, interleaved, [&](auto lpr, auto il) {
      hipLaunchKernelGGL((norm_rotate_kernel<T, decltype(lpr)::value, decltype(il)::value>),
                         dim3(static_cast<unsigned>(a.side[0].blocks + a.side[1].blocks)),
                         dim3(kThreads), 0, as_stream(stream), a);
      return check_launch("moba_norm_rotate");
    });
  });
}

extern "C" size_t moba_norm_rotate_bwd_workspace_size(int64_t head_dim) {
  return sizeof(float) * static_cast<size_t>(moba::kMaxBlocks * (head_dim > 0 ? head_dim : 0));
}

extern "C" int moba_norm_rotate_bwd(const void* dq_out, const void* dk_out, const void* q,
                                    const void* k, void* dq, void* dk, void* dq_weight,
                                    void* dk_weight, const float* cos_table,
                                    const float* sin_table, const int32_t* positions,
                                    const void* q_weight, const void* k_weight, int64_t batch,
                                    int64_t seq_len, int64_t h_q, int64_t h_kv, int64_t head_dim,
                                    const int64_t* strides, int64_t rotary, int64_t table_len,
                                    int interleaved, double eps, int dtype, int weight_dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace moba;
  int st = check(batch, seq_len, h_q, h_kv, head_dim, rotary, table_len, cos_table, sin_table,
                 dtype, weight_dtype);
  if (!st) st = check_rows({dq_out, dk_out, q, k, dq, dk}, strides, dtype);
  if (st) return st;
  if ((q_weight != nullptr) != (dq_weight != nullptr) ||
      (k_weight != nullptr) != (dk_weight != nullptr))
    return fail(MOBA_ERR_INVALID, "a norm weight and its gradient go together");
  RotArgs a = make_args(q, k, dq, dk, cos_table, sin_table, positions, q_weight, k_weight, batch,
                        seq_len, h_q, h_kv, strides, rotary, table_len, eps,
                        weight_dtype);
  a.side[0].dy = dq_out;
  a.side[1].dy = dk_out;
  set_blocks(&a, head_dim);
  if (q_weight || k_weight) {
    if (!workspace || workspace_bytes < moba_norm_rotate_bwd_workspace_size(head_dim))
      return fail(MOBA_ERR_WORKSPACE, "norm_rotate_bwd workspace too small");
    a.side[0].partial = static_cast<float*>(workspace);
    a.side[1].partial = a.side[0].partial + a.side[0].blocks * head_dim;
  }
  st = MOBA_DISPATCH_DTYPE(dtype, T, [&] {
    return with_lanes(head_dim, interleaved, [&](auto lpr, auto il) {
      hipLaunchKernelGGL((norm_rotate_bwd_kernel<T, decltype(lpr)::value, decltype(il)::value>),
                         dim3(static_cast<unsigned>(a.side[0].blocks + a.side[1].blocks)),
                         dim3(kThreads), 0, as_stream(stream), a);
      return check_launch("moba_norm_rotate_bwd");
    });
  });
  if (st || !(q_weight || k_weight)) return st;
  return MOBA_DISPATCH_DTYPE(weight_dtype, W, [&] {
    hipLaunchKernelGGL(norm_weight_kernel<W>, dim3(static_cast<unsigned>(head_dim / 16), 2),
                       dim3(1024), 0, as_stream(stream), a.side[0].partial, a.side[0].blocks,
                       static_cast<W*>(dq_weight), a.side[1].partial, a.side[1].blocks,
                       static_cast<W*>(dk_weight), static_cast<int>(head_dim));
    return check_launch("moba_norm_rotate_bwd (weights)");
  });
}
