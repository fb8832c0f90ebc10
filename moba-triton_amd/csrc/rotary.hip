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
// dw: every workgroup sums its rows in float32 (tens of rows per lane), its
// lanes meet in LDS in a fixed order, and a second kernel adds the
// workgroups' sums in float64 in order: the result depends on the shape only.
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
  int slices;         // lane groups that share a token's heads
  float* partial;     // backward: dw sums [workgroups, D]
  int blocks;         // workgroups of this side
};

struct RotArgs {
  RotSide side[2];  // queries, keys
  const float* cosv;
  const float* sinv;
  const int32_t* positions;  // [batch * seq], or null: 0, 1, .. in each row
  int64_t tokens, seq, table_len;
  int rotary, interleaved, w_f32;
  float eps;
};

// Workgroups' sizes and the rows a lane group holds at a time.
constexpr int kThreads = 256;
constexpr int kRows = 4;

template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads) norm_rotate_kernel(RotArgs a) {
  constexpr int D = 16 * LPR;
  const bool second = static_cast<int>(blockIdx.x) >= a.side[0].blocks;
  const RotSide s = a.side[second];
  const int64_t block = static_cast<int64_t>(blockIdx.x) - (second ? a.side[0].blocks : 0);
  const int lane = threadIdx.x % LPR;
  const int64_t group = (block * kThreads + threadIdx.x) / LPR;
  const int64_t tok = group / s.slices;
  if (tok >= a.tokens) return;  // whole lane groups
  const int slice = static_cast<int>(group - tok * s.slices);
  const RotLane rl = rot_lane(lane, a.rotary, a.interleaved);
  float c[8], sn[8];
  rot_turn(rl, a.cosv, a.sinv, a.rotary,
           a.positions ? a.positions[tok] : static_cast<int32_t>(tok % a.seq), a.table_len, c, sn);
  float w[16];
  if (s.w) load16<T>(s.w, a.w_f32, rl, w);
  const T* x = static_cast<const T*>(s.x) + (tok / a.seq) * s.sb + (tok % a.seq) * s.ss;
  T* y = static_cast<T*>(s.y) + tok * s.heads * D;
  for (int h0 = slice; h0 < s.heads; h0 += kRows * s.slices) {
    RawRow<T> raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int h = h0 + i * s.slices;
      raw[i].load(x + static_cast<int64_t>(h < s.heads ? h : h0) * s.sh, rl);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int h = h0 + i * s.slices;
      if (h >= s.heads) break;
      float v[16];
      raw[i].widen(v);
      if (s.w) {
        const float r = rsqrtf(row_sum<LPR>(square_sum(v)) * (1.f / D) + a.eps);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * r * w[e];
      }
      rotate16(rl, c, sn, v);
      raw[i].narrow(v);
      raw[i].store(y + static_cast<int64_t>(h) * D, rl);
    }
  }
}

// dx, and this workgroup's share of dw. Workgroups of a side stride over its
// lane groups' work, so the number of partial sums is bounded.
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads) norm_rotate_bwd_kernel(RotArgs a) {
  constexpr int D = 16 * LPR;
  constexpr int kGroups = kThreads / LPR;  // lane groups of the workgroup
  constexpr int R = 2;                     // rows in flight: x and dy of each
  __shared__ float sums[kThreads / 64][D];
  const bool second = static_cast<int>(blockIdx.x) >= a.side[0].blocks;
  const RotSide s = a.side[second];
  const int64_t block = static_cast<int64_t>(blockIdx.x) - (second ? a.side[0].blocks : 0);
  const int lane = threadIdx.x % LPR;
  const RotLane rl = rot_lane(lane, a.rotary, a.interleaved);
  float w[16], dw[16];
  if (s.w) load16<T>(s.w, a.w_f32, rl, w);
#pragma unroll
  for (int e = 0; e < 16; ++e) dw[e] = 0.f;
  const int64_t work = a.tokens * s.slices;
  for (int64_t group = block * kGroups + threadIdx.x / LPR; group < work;
       group += static_cast<int64_t>(s.blocks) * kGroups) {
    const int64_t tok = group / s.slices;
    const int slice = static_cast<int>(group - tok * s.slices);
    float c[8], sn[8];
    rot_turn(rl, a.cosv, a.sinv, a.rotary,
             a.positions ? a.positions[tok] : static_cast<int32_t>(tok % a.seq), a.table_len, c, sn);
    const T* x = static_cast<const T*>(s.x) + (tok / a.seq) * s.sb + (tok % a.seq) * s.ss;
    const T* dy = static_cast<const T*>(s.dy) + tok * s.heads * D;
    T* dx = static_cast<T*>(s.y) + tok * s.heads * D;
    for (int h0 = slice; h0 < s.heads; h0 += R * s.slices) {
      RawRow<T> rx[R], rg[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int h = h0 + i * s.slices < s.heads ? h0 + i * s.slices : h0;
        rg[i].load(dy + static_cast<int64_t>(h) * D, rl);
        if (s.w) rx[i].load(x + static_cast<int64_t>(h) * s.sh, rl);
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int h = h0 + i * s.slices;
        if (h >= s.heads) break;
        float g[16];
        rg[i].widen(g);
        unrotate16(rl, c, sn, g);
        if (s.w) {
          float v[16];
          rx[i].widen(v);
          const float r = rsqrtf(row_sum<LPR>(square_sum(v)) * (1.f / D) + a.eps);
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            v[e] *= r;
            dw[e] = fmaf(g[e], v[e], dw[e]);
            g[e] *= w[e];
            dot = fmaf(g[e], v[e], dot);
          }
          dot = row_sum<LPR>(dot) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 16; ++e) g[e] = r * (g[e] - v[e] * dot);
        }
        rg[i].narrow(g);
        rg[i].store(dx + static_cast<int64_t>(h) * D, rl);
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
// 16 threads per feature take every 16th workgroup and meet by shuffles.
// grid (D / 16, 2).
template <typename W>
__global__ void __launch_bounds__(256)
norm_weight_kernel(const float* __restrict__ pq, int nq, W* __restrict__ dwq,
                   const float* __restrict__ pk, int nk, W* __restrict__ dwk, int D) {
  const float* p = blockIdx.y ? pk : pq;
  const int n = blockIdx.y ? nk : nq;
  W* out = blockIdx.y ? dwk : dwq;
  if (!out) return;
  // Lanes along the features (64-byte reads), partial sums through LDS.
  __shared__ double part[16][17];
  const int d = threadIdx.x & 15, j = threadIdx.x >> 4;
  const int feature = blockIdx.x * 16 + d;
  double t = 0.0;
#pragma unroll 4
  for (int i = j; i < n; i += 16) t += static_cast<double>(p[static_cast<int64_t>(i) * D + feature]);
  part[j][d] = t;
  __syncthreads();
  if (j) return;
  for (int i = 1; i < 16; ++i) t += part[i][d];
  Elem<W>::store(out, feature, static_cast<float>(t));
}

int check(int64_t batch, int64_t seq, int64_t h_q, int64_t h_kv, int64_t D, int64_t rotary,
          int64_t table_len, const void* cosv, const void* sinv, int dtype, int w_dtype) {
  if (batch <= 0 || seq <= 0 || h_q <= 0 || h_kv <= 0)
    return fail(MOBA_ERR_INVALID, "non-positive shape argument");
  const int st = check_rotary(D, rotary, table_len, cosv, sinv, dtype, w_dtype);
  if (st) return st;
  if (batch * seq > (int64_t(1) << 31) - 1)
    return fail(MOBA_ERR_UNSUPPORTED, "norm_rotate: more than 2^31 - 1 tokens");
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

// Lane groups per token: one group holds kRows heads at a time; a call with
// few rows takes a group for each head instead, so the rows are in flight at
// once on an otherwise idle chip.
int slices_of(int64_t tokens, int heads) {
  const int few = (heads + kRows - 1) / kRows;
  return tokens * heads <= 1 << 15 ? heads : few;
}

template <typename F>
int with_lanes(int64_t D, F&& go) {
  switch (D) {
    case 32: return go(std::integral_constant<int, 2>{});
    case 64: return go(std::integral_constant<int, 4>{});
    case 128: return go(std::integral_constant<int, 8>{});
    case 256: return go(std::integral_constant<int, 16>{});
    case 512: return go(std::integral_constant<int, 32>{});
    default: return go(std::integral_constant<int, 64>{});
  }
}

// Workgroups of one side of the backward: at most kBwdBlocks in all, so that
// a lane sums tens of rows before it meets the others.
constexpr int64_t kBwdBlocks = 2048;
int64_t bwd_blocks(int64_t tokens, int slices, int64_t D, int64_t share) {
  const int64_t need = cdiv(tokens * slices, kThreads / (D / 16));
  return need < share ? need : share;
}

RotArgs make_args(const void* q, const void* k, void* yq, void* yk, const float* cosv,
                  const float* sinv, const int32_t* positions, const void* wq, const void* wk,
                  int64_t batch, int64_t seq, int64_t h_q, int64_t h_kv, const int64_t* strides,
                  int64_t rotary, int64_t table_len, int interleaved, double eps, int w_dtype) {
  RotArgs a;
  a.side[0] = {q, nullptr, yq, wq, strides[0], strides[1], strides[2], static_cast<int>(h_q),
               slices_of(batch * seq, static_cast<int>(h_q)), nullptr, 0};
  a.side[1] = {k, nullptr, yk, wk, strides[3], strides[4], strides[5], static_cast<int>(h_kv),
               slices_of(batch * seq, static_cast<int>(h_kv)), nullptr, 0};
  a.cosv = cosv;
  a.sinv = sinv;
  a.positions = positions;
  a.tokens = batch * seq;
  a.seq = seq;
  a.table_len = table_len;
  a.rotary = static_cast<int>(rotary);
  a.interleaved = interleaved;
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
                        batch, seq_len, h_q, h_kv, strides, rotary, table_len, interleaved, eps,
                        weight_dtype);
  for (RotSide& s : a.side) {
    const int64_t blocks = cdiv(a.tokens * s.slices, kThreads / (head_dim / 16));
    if (blocks > (1 << 30)) return fail(MOBA_ERR_UNSUPPORTED, "norm_rotate: too many rows");
    s.blocks = static_cast<int>(blocks);
  }
  return MOBA_DISPATCH_DTYPE(dtype, T, [&] {
    return with_lanes(head_dim, [&](auto lpr) {
      hipLaunchKernelGGL((norm_rotate_kernel<T, decltype(lpr)::value>),
                         dim3(static_cast<unsigned>(a.side[0].blocks + a.side[1].blocks)),
                         dim3(kThreads), 0, as_stream(stream), a);
      return check_launch("moba_norm_rotate");
    });
  });
}

extern "C" size_t moba_norm_rotate_bwd_workspace_size(int64_t head_dim) {
  return sizeof(float) * static_cast<size_t>(moba::kBwdBlocks * (head_dim > 0 ? head_dim : 0));
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
                        seq_len, h_q, h_kv, strides, rotary, table_len, interleaved, eps,
                        weight_dtype);
  a.side[0].dy = dq_out;
  a.side[1].dy = dk_out;
  // Each side's share of the workgroups goes by its rows.
  int64_t share = kBwdBlocks * h_q / (h_q + h_kv);
  share = share < 1 ? 1 : (share < kBwdBlocks ? share : kBwdBlocks - 1);
  a.side[0].blocks = static_cast<int>(bwd_blocks(a.tokens, a.side[0].slices, head_dim, share));
  a.side[1].blocks =
      static_cast<int>(bwd_blocks(a.tokens, a.side[1].slices, head_dim, kBwdBlocks - share));
  if (q_weight || k_weight) {
    if (!workspace || workspace_bytes < moba_norm_rotate_bwd_workspace_size(head_dim))
      return fail(MOBA_ERR_WORKSPACE, "norm_rotate_bwd workspace too small");
    a.side[0].partial = static_cast<float*>(workspace);
    a.side[1].partial = a.side[0].partial + a.side[0].blocks * head_dim;
  }
  st = MOBA_DISPATCH_DTYPE(dtype, T, [&] {
    return with_lanes(head_dim, [&](auto lpr) {
      hipLaunchKernelGGL((norm_rotate_bwd_kernel<T, decltype(lpr)::value>),
                         dim3(static_cast<unsigned>(a.side[0].blocks + a.side[1].blocks)),
                         dim3(kThreads), 0, as_stream(stream), a);
      return check_launch("moba_norm_rotate_bwd");
    });
  });
  if (st || !(q_weight || k_weight)) return st;
  return MOBA_DISPATCH_DTYPE(weight_dtype, W, [&] {
    hipLaunchKernelGGL(norm_weight_kernel<W>, dim3(static_cast<unsigned>(head_dim / 16), 2),
                       dim3(256), 0, as_stream(stream), a.side[0].partial, a.side[0].blocks,
                       static_cast<W*>(dq_weight), a.side[1].partial, a.side[1].blocks,
                       static_cast<W*>(dk_weight), static_cast<int>(head_dim));
    return check_launch("moba_norm_rotate_bwd (weights)");
  });
}
