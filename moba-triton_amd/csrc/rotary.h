// A head's row in registers: 16 features per lane, norm and rotation.
#pragma once

#include <type_traits>

#include "common.h"

namespace moba {

// Which features a lane of a row holds: [lo, lo + 8) and [hi, hi + 8). Halves:
// the lanes of the rotated part hold pairs (lo + i, hi + i), hi = lo +
// rotary / 2. Neighbours: 16 consecutive features, pairs (2i, 2i + 1). The
// lanes behind the rotated part hold 16 consecutive features each.
struct RotLane {
  int lo, hi;
  bool turn;       // rotated
  int angle;       // first of the lane's 8 angles
};

__device__ inline RotLane rot_lane(int lane, int rotary, int interleaved) {
  RotLane r;
  const bool in = 16 * lane < rotary;
  const bool halves = in && !interleaved;
  r.lo = halves ? 8 * lane : 16 * lane;
  r.hi = halves ? rotary / 2 + 8 * lane : 16 * lane + 8;
  r.turn = in;
  r.angle = 8 * lane;
  return r;
}

// The lane's cosines and sines of position `pos`. A position outside the
// table gives NaN, and so do the rotated features: nothing outside the table is
// read.
__device__ inline void rot_turn(const RotLane& r, const float* cosv, const float* sinv, int rotary,
                                int64_t pos, int64_t table_len, float (&c)[8], float (&s)[8]) {
  const bool ok = pos >= 0 && pos < table_len;
  if (r.turn && ok) {
    const int64_t at = pos * (rotary / 2) + r.angle;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(cosv + at + i);
      const float4 sv = *reinterpret_cast<const float4*>(sinv + at + i);
      c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
      s[i] = sv.x; s[i + 1] = sv.y; s[i + 2] = sv.z; s[i + 3] = sv.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = r.turn ? NAN : 1.f;
      s[i] = r.turn ? NAN : 0.f;
    }
  }
}

// v[0, 8) are the features from lo, v[8, 16) those from hi. By selects, not
// branches: lanes that are not rotated keep their values whatever they are.
// IL: neighbouring pairs (a template: a branch would let the compiler index
// the row by it, in scratch memory).
template <bool IL>
__device__ inline void rotate16(const RotLane& r, const float (&c)[8], const float (&s)[8],
                                float (&v)[16]) {
  const bool on = r.turn;
  if constexpr (IL) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1];
      const float x = a * c[i] - b * s[i], y = b * c[i] + a * s[i];
      v[2 * i] = on ? x : a;
      v[2 * i + 1] = on ? y : b;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = v[i], b = v[8 + i];
      const float x = a * c[i] - b * s[i], y = b * c[i] + a * s[i];
      v[i] = on ? x : a;
      v[8 + i] = on ? y : b;
    }
  }
}

template <bool IL>
__device__ inline void unrotate16(const RotLane& r, const float (&c)[8], const float (&s)[8],
                                  float (&v)[16]) {
  float n[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = -s[i];
  rotate16<IL>(r, c, n, v);
}

__device__ inline float square_sum(const float (&v)[16]) {
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) t = fmaf(v[e], v[e], t);
  return t;
}

// Sum over the LPR adjacent lanes of a row.
template <int LPR>
__device__ inline float row_sum(float t) {
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) t += __shfl_xor(t, off);
  return t;
}

typedef uint32_t rot_u32x4 __attribute__((ext_vector_type(4)));

// A lane's 16 elements as they lie in memory.
template <typename T>
struct RawRow {
  static constexpr int P = static_cast<int>(sizeof(T)) / 2;  // 16-byte pieces per 8 elements
  rot_u32x4 piece[2 * P];
  __device__ void load(const T* row, const RotLane& r) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      piece[i] = *reinterpret_cast<const rot_u32x4*>(row + r.lo + i * (8 / P));
      piece[P + i] = *reinterpret_cast<const rot_u32x4*>(row + r.hi + i * (8 / P));
    }
  }
  __device__ void store(T* row, const RotLane& r) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      *reinterpret_cast<rot_u32x4*>(row + r.lo + i * (8 / P)) = piece[i];
      *reinterpret_cast<rot_u32x4*>(row + r.hi + i * (8 / P)) = piece[P + i];
    }
  }
  __device__ void widen(float (&v)[16]) const {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = element(e);
  }
  __device__ float element(int e) const {
    if constexpr (sizeof(T) == 4) {
      return u2f(piece[e >> 2][e & 3]);
    } else {
      const uint32_t u = piece[e >> 3][(e & 7) >> 1];
      if constexpr (std::is_same<T, bf16_t>::value) {
        return u2f(e & 1 ? u & 0xffff0000u : u << 16);
      } else {
        return static_cast<float>(
            __builtin_bit_cast(_Float16, static_cast<uint16_t>(e & 1 ? u >> 16 : u)));
      }
    }
  }
  // Rounded to nearest even by the hardware conversions.
  __device__ void narrow(const float (&v)[16]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 16; ++e) piece[e >> 2][e & 3] = f2u(v[e]);
    } else {
      typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        uint32_t u;
        if constexpr (std::is_same<T, bf16_t>::value) {
          typedef __bf16 h2 __attribute__((ext_vector_type(2)));
          u = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{v[e], v[e + 1]}, h2));
        } else {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          u = __builtin_bit_cast(
              uint32_t, h2{static_cast<_Float16>(v[e]), static_cast<_Float16>(v[e + 1])});
        }
        piece[e >> 3][(e & 7) >> 1] = u;
      }
    }
  }
};

// A lane's 16 elements of a vector of D in float32 (f32) or T.
template <typename T>
__device__ inline void load16(const void* p, int f32, const RotLane& r, float (&v)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int64_t at = e < 8 ? r.lo + e : r.hi + e - 8;
    v[e] = f32 ? static_cast<const float*>(p)[at] : Elem<T>::load(static_cast<const T*>(p), at);
  }
}

inline bool on_16_bytes(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Host checks shared by the calls that norm and rotate.
int check_rotary(int64_t head_dim, int64_t rotary, int64_t table_len, const void* cosv,
                 const void* sinv, int dtype, int weight_dtype);

}  // namespace moba
