// gated_device.h -- operand types and 16-byte pieces of the gated feed-forward kernels (gated.hip).
//
// Everything moves in 16-byte pieces of a row: E = 8 f16 / bf16 or 4 f32 elements.  A UNIT is 64 bytes of a row = four pieces,
// one for each 16-lane quarter kg of a wave: lane (j = lane & 15, kg = lane >> 4) holds piece kg of its row's unit.  That is the
// operand layout of v_mfma_f32_16x16x32_{f16,bf16} (one instruction a unit) and, with the contraction index taken as
// k = 16 u + 4 kg + m, of four v_mfma_f32_16x16x4_f32: both operands use the same order, so the sum does not see it.
// Accumulators: lane (j, kg), register r = row 4 kg + r, column j.
#pragma once
#include "gfn_common.h"

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

enum { GATED_SILU = 0, GATED_GELU = 1, GATED_RELU = 2, GATED_SIGMOID = 3 };

template <typename T>
struct Piece {
  static constexpr int E = 16 / (int)sizeof(T);
};

__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 c, __bf16*) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 c, _Float16*) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 c, float*) {
#pragma unroll
  for (int m = 0; m < 4; m++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a)[m], __builtin_bit_cast(f32x4, b)[m], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ u32x4 load16(const void* p) {  // rows of odd width start at any element: no alignment is assumed
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// Piece c (elements c E .. c E + E - 1) of a row of `k` elements, zeros behind its end; nothing outside the row is read.  In two steps,
// so that a piece can be requested long before it is looked at: the piece that the row's end cuts is REQUESTED as the row's last 16
// bytes, and CUT (shifted down by what it holds too early: the same shift in every lane) where it is used.
template <typename T>
__device__ __forceinline__ u32x4 piece_request(const T* row, int c, int k) {
  constexpr int E = Piece<T>::E;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (c * E >= k) return v;
  if (k >= E) return load16(row + (c * E + E <= k ? c * E : k - E));
  T e[E];
#pragma unroll
  for (int i = 0; i < E; i++) e[i] = i < k ? row[i] : (T)0.f;
  __builtin_memcpy(&v, e, 16);
  return v;
}
// the piece that the end of a row of `k` elements cuts, or -1; the same in every lane
template <typename T>
__device__ __forceinline__ int cut_piece(int k) {
  constexpr int E = Piece<T>::E;
  return k > E && k % E ? k / E : -1;
}
template <typename T>
__device__ __forceinline__ u32x4 piece_shift(u32x4 w, int k) {
  constexpr int E = Piece<T>::E;
  const int left = k % E;
  u32x4 v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 3; i++)  // element i of the piece = element i + E - left of the row's last E
      v[i] = i < left ? (left == 3 ? w[i + 1] : left == 2 ? w[(i + 2) & 3] : w[3]) : 0u;
    v[3] = 0u;
  } else {
    typedef unsigned __int128 u128;
    const u128 s = __builtin_bit_cast(u128, w) >> (16 * (E - left));
    v = __builtin_bit_cast(u32x4, s);
  }
  return v;
}
template <typename T>
__device__ __forceinline__ u32x4 row_piece(const T* row, int c, int k) {
  const u32x4 w = piece_request(row, c, k);
  return c == cut_piece<T>(k) ? piece_shift<T>(w, k) : w;
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, int left, const float (&v)[N]) {
  using Row = __attribute__((ext_vector_type(N))) T;
  Row e;
#pragma unroll
  for (int i = 0; i < N; i++) e[i] = (T)v[i];
  if (left >= N) {
    if constexpr (sizeof(Row) == 8) __builtin_memcpy(p, &e, 8);
#pragma unroll
    for (int c = 0; c < (int)sizeof(Row) / 16; c++) {
      using Rows = __attribute__((ext_vector_type(sizeof(Row) / 4))) uint32_t;
      const Rows r = __builtin_bit_cast(Rows, e);
      const u32x4 q = {r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]};
      __builtin_memcpy(reinterpret_cast<char*>(p) + 16 * c, &q, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < left) p[i] = e[i];
  }
}

// 1 / (1 + exp(-z)).  For 16-bit results the hardware's exp2 and reciprocal as they are (2^-22 of the value: far below the result's rounding);
// EXACT (f32): the argument's rounding put back (exp2(t + r) = exp2(t) (1 + r ln 2)) and one Newton step on the reciprocal.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
  const float t = z * -1.44269504088896340736f;
  float e = __builtin_amdgcn_exp2f(t);
  if constexpr (!EXACT) return __builtin_amdgcn_rcpf(1.f + e);
  e = __builtin_fmaf(e, __builtin_fmaf(z, -1.44269504088896340736f, -t) * 0.693147180559945309417f, e);
  const float d = 1.f + e, r = __builtin_amdgcn_rcpf(d);
  const float s = __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r);
  return t > 126.f ? 0.f : (t < -126.f ? 1.f : s);  // where exp2 over- or underflows the two steps would meet inf - inf
}

// Phi(z) = erfc(-z / sqrt 2) / 2, and gauss = exp(-z^2 / 2), which its derivative needs as well.  With x = |z| / sqrt 2 and
// t = 1 / (1 + c x), erfc(x) = t exp(-x^2) P(t): exp(x^2) erfc(x) / t is smooth on (0, 1] and P is its least-largest-relative-error
// polynomial, fitted to 64-bit values.  EXACT (f32): degree 8, c = 0.4, 1.3e-7 of the tail, and 2.2e-7 with the rounding of its sums;
// else degree 7, c = 0.46, 7.6e-7.
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float z, float& gauss) {
  gauss = __builtin_amdgcn_exp2f(-0.72134752044448170368f * z * z);  // -z^2 / 2 / ln 2
  const float x = 0.70710678118654752440f * __builtin_fabsf(z);
  float t, p;
  if constexpr (EXACT) {
    t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f, x, 1.f));
    p = __builtin_fmaf(0.0502589586f, t, -0.182889897f);
    p = __builtin_fmaf(p, t, 0.169068453f);
    p = __builtin_fmaf(p, t, -0.00559473326f);
    p = __builtin_fmaf(p, t, 0.141426169f);
    p = __builtin_fmaf(p, t, 0.168543132f);
    p = __builtin_fmaf(p, t, 0.207842577f);
    p = __builtin_fmaf(p, t, 0.225669603f);
    p = __builtin_fmaf(p, t, 0.225675862f);
  } else {
    t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.46f, x, 1.f));
    p = __builtin_fmaf(0.0677144445f, t, -0.226629622f);
    p = __builtin_fmaf(p, t, 0.16919146f);
    p = __builtin_fmaf(p, t, 0.0526103041f);
    p = __builtin_fmaf(p, t, 0.186847901f);
    p = __builtin_fmaf(p, t, 0.231181864f);
    p = __builtin_fmaf(p, t, 0.259557267f);
    p = __builtin_fmaf(p, t, 0.259527059f);
  }
  const float tail = 0.5f * p * t * gauss;
  return z < 0.f ? tail : 1.f - tail;
}

// v[i] = act(g[i]) u[i] for eight values.  A NaN stays one.
template <int ACT, bool EXACT, typename F, typename U>
__device__ __forceinline__ void gated8(F g, U u, float (&v)[8]) {
  switch (ACT) {
    case GATED_SILU:
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = g(i) * sigmoid<EXACT>(g(i)) * u(i);
      break;
    case GATED_GELU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float gauss;
        v[i] = g(i) * normal_cdf<EXACT>(g(i), gauss) * u(i);
      }
      break;
    case GATED_RELU:
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = (g(i) < 0.f ? 0.f : g(i)) * u(i);
      break;
    default:
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = sigmoid<EXACT>(g(i)) * u(i);
  }
}
// dg[i] = d[i] u[i] act'(g[i]), du[i] = d[i] act(g[i]).  A NaN stays one.
template <int ACT, bool EXACT, typename F, typename U>
__device__ __forceinline__ void gated8_grad(F g, U u, const float (&d)[8], float (&dg)[8], float (&du)[8]) {
  switch (ACT) {
    case GATED_SILU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float s = sigmoid<EXACT>(g(i)), a = g(i) * s;
        dg[i] = (d[i] * u(i) * __builtin_fmaf(a, 1.f - s, s));
        du[i] = (d[i] * a);
      }
      break;
    case GATED_GELU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float gauss;
        const float cdf = normal_cdf<EXACT>(g(i), gauss);
        dg[i] = (d[i] * u(i) * __builtin_fmaf(g(i) * 0.39894228040143267794f, gauss, cdf));
        du[i] = (d[i] * (g(i) * cdf));
      }
      break;
    case GATED_RELU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        dg[i] = g(i) > 0.f ? d[i] * u(i) : (g(i) <= 0.f ? 0.f : g(i));
        du[i] = (d[i] * (g(i) < 0.f ? 0.f : g(i)));
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float s = sigmoid<EXACT>(g(i));
        dg[i] = (d[i] * u(i) * (s * (1.f - s)));
        du[i] = (d[i] * s);
      }
  }
}

}  // namespace
