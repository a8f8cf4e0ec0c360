// What the kernels of the dense layer (dense_tcgen05.cuh, dense_rows.cuh) share: the two 16-bit types, the
// activations and their slopes, and the plan by which a product is split over its contraction.
//
//   y = r + act(z),  z = x W^T + b          x [M, K], W [N, K]
//   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum over rows of dz
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace strata {

enum DenseAct : int { ACT_NONE = 0, ACT_GELU = 1, ACT_GELU_TANH = 2, ACT_SILU = 3, ACT_RELU = 4, ACT_COUNT = 5,
                      ACT_ANY = -1 };

// Two values of a 16-bit type in a word; sums, products and activations are all fp32, a value is rounded once, when it
// is stored.
template <typename T> struct Pair16;
template <> struct Pair16<__nv_bfloat16> {
  static constexpr uint32_t UMMA_FORMAT = 1;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
  static __device__ __forceinline__ float lo(uint32_t v) { return bf16_lo(v); }
  static __device__ __forceinline__ float hi(uint32_t v) { return bf16_hi(v); }
};
template <> struct Pair16<__half> {
  static constexpr uint32_t UMMA_FORMAT = 0;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float lo(uint32_t v) {
    return __low2float(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ float hi(uint32_t v) {
    return __high2float(*reinterpret_cast<const __half2*>(&v));
  }
};
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The slope's Phi: the normal distribution's upper tail Q(a) = 1 - Phi(a), a >= 0, by formula 7.1.26 of Abramowitz and
// Stegun (erf to 1.5e-7) with x = a / sqrt(2); e = exp(-a^2 / 2).
constexpr float GELU_P = 0.3275911f * 0.70710678118654752f;
constexpr float GELU_C1 = 0.5f * 0.254829592f, GELU_C2 = 0.5f * -0.284496736f, GELU_C3 = 0.5f * 1.421413741f,
                GELU_C4 = 0.5f * -1.453152027f, GELU_C5 = 0.5f * 1.061405429f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float GELU_K0 = 0.7978845608028654f, GELU_K1 = 0.044715f;   // sqrt(2 / pi)

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// x / (1 + 2^v) of a pair with one reciprocal for both: 1 / a = b / (a b). 2^v must stay below 2^63, and v may not be
// NaN: it would reach the other value. b times the reciprocal comes first: x b may leave fp32 where x / a does not.
__device__ __forceinline__ uint64_t dense_sigmoid_pair(uint64_t x, uint64_t v) {
  float v0, v1, d0, d1;
  unpack2(v, v0, v1);
  unpack2(fadd2(pack2(fast_exp2(v0), fast_exp2(v1)), pack2(1.f, 1.f)), d0, d1);
  const float r = fast_rcp(d0 * d1);
  return fmul2(x, fmul2(pack2(d1, d0), pack2(r, r)));
}

// The forward pass's gelu: max(x, 0) - a Phi(-a), a = |x|, with Phi(-a) = 2^q(a): the logarithm of the tail is smooth,
// so a polynomial in a has it over all magnitudes at once, nothing cancels, and one special-function instruction a
// value is enough (x / (1 + e^-L(x)) with a fitted logit takes three a pair, and an erf of absolute accuracy has
// nothing right in the tail). Fitted for the least largest error, relative to |gelu| where a type can see that (half
// steps: bf16 3.9e-3, fp16 4.9e-4):
//   bf16   8.1e-5 for x > -4, 2.2e-4 to -6, 3.8e-3 to -8, 5 % to -9; below -10, where |gelu| < 1e-22, the right order
//   fp16   6.3e-6 for x > -4, off by 4e-10 at most below (half of the smallest step: 3e-8)
// 262144 x 2048, K = 512, bf16: 465 us with seven coefficients, 493 with nine (one fit for both types), 495 with a
// fitted logit of five. (coefficients: in -a, which stops at FAR)
template <typename T> struct GeluFit;
template <> struct GeluFit<__nv_bfloat16> {
  static constexpr int N = 7;
  static constexpr float FAR = -13.f;
  static __device__ constexpr float c(int i) {
    constexpr float k[N] = {-1.00011623f,   1.14947224f,     -0.462817311f,  0.0499514751f,
                            0.00675397133f, 0.000538877153f, 1.86031939e-05f};
    return k[i];
  }
};
template <> struct GeluFit<__half> {
  static constexpr int N = 7;
  static constexpr float FAR = -6.5f;
  static __device__ constexpr float c(int i) {
    constexpr float k[N] = {-1.00000763f,   1.15103662f,     -0.459170461f,  0.0530517921f,
                            0.00794225838f, 0.000748418213f, 3.24445282e-05f};
    return k[i];
  }
};

// act(x) of a pair. silu: x / (1 + e^-x). gelu_tanh: x / (1 + e^-v), v = 2 k0 (x + k1 x^3), which is its 0.5 x (1 +
// tanh(v / 2)): the hardware's tanh, right to 2^-11 of itself, is two instructions a pair instead of three but leaves
// 1 + tanh little on the negative side (20 % off at -3). 262144 x 2048, K = 512: 447 us against 428, with a residual
// 550 against 519. Below -40 and -7.5 they keep those points' values, 2e-16 and 4e-18.
template <typename T, int ACT>
__device__ __forceinline__ uint64_t dense_act_pair(uint64_t x) {
  float a, b;
  unpack2(x, a, b);
  if constexpr (ACT == ACT_GELU_TANH) {
    constexpr float C0 = -2.f * LOG2E * GELU_K0, C1 = C0 * GELU_K1;
    x = pack2(max_nan(a, -7.5f), max_nan(b, -7.5f));
    const uint64_t e = pack2(fmaxf(a, -7.5f), fmaxf(b, -7.5f));       // (no NaN)
    return dense_sigmoid_pair(x, fmul2(e, ffma2(fmul2(e, e), pack2(C1, C1), pack2(C0, C0))));
  } else if constexpr (ACT == ACT_GELU) {
    using F = GeluFit<T>;      // (a NaN is left to the first term)
    const uint64_t n = pack2(fmaxf(-fabsf(a), F::FAR), fmaxf(-fabsf(b), F::FAR));
    uint64_t q = pack2(F::c(F::N - 1), F::c(F::N - 1));
#pragma unroll
    for (int i = F::N - 2; i >= 0; --i) q = ffma2(q, n, pack2(F::c(i), F::c(i)));
    float q0, q1;
    unpack2(q, q0, q1);
    return ffma2(n, pack2(fast_exp2(q0), fast_exp2(q1)), pack2(max_nan(a, 0.f), max_nan(b, 0.f)));
  } else if constexpr (ACT == ACT_SILU) {
    x = pack2(max_nan(a, -40.f), max_nan(b, -40.f));
    return dense_sigmoid_pair(x, fmul2(pack2(fmaxf(a, -40.f), fmaxf(b, -40.f)), pack2(-LOG2E, -LOG2E)));
  } else if constexpr (ACT == ACT_RELU) {
    return pack2(max_nan(a, 0.f), max_nan(b, 0.f));
  } else {
    return x;
  }
}

template <typename T, int ACT, int N>
__device__ __forceinline__ void dense_act_all(uint64_t (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = dense_act_pair<T, ACT>(v[i]);
}
// `act` is the same for the whole launch.
template <typename T, int N>
__device__ __forceinline__ void dense_act(int act, uint64_t (&v)[N]) {
  switch (act) {
    case ACT_GELU: dense_act_all<T, ACT_GELU>(v); break;
    case ACT_GELU_TANH: dense_act_all<T, ACT_GELU_TANH>(v); break;
    case ACT_SILU: dense_act_all<T, ACT_SILU>(v); break;
    case ACT_RELU: dense_act_all<T, ACT_RELU>(v); break;
    default: break;
  }
}

// act'(z). A stored z may be infinite (fp16): the slope is then that of a far z, 0 or 1 to 1e-11; NaN stays NaN. 1 - s
// of s = 1 / (1 + e) is taken as e s: the difference would lose the digits that z s (1 - s) multiplies up.
template <int ACT>
__device__ __forceinline__ float dense_slope(float z) {
  if constexpr (ACT == ACT_NONE) return 1.f;
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  constexpr float FAR = ACT == ACT_GELU_TANH ? 8.f : 30.f;             // (e stays finite)
  z = z > FAR ? FAR : (z < -FAR ? -FAR : z);
  if constexpr (ACT == ACT_GELU) {
    const float a = fabsf(z), t = fast_rcp(fmaf(a, GELU_P, 1.f)), e = fast_exp2(z * z * (-0.5f * LOG2E));
    const float q = (fmaf(fmaf(fmaf(fmaf(GELU_C5, t, GELU_C4), t, GELU_C3), t, GELU_C2), t, GELU_C1) * t) * e;
    return fmaf(z * 0.3989422804014327f, e, z >= 0.f ? 1.f - q : q);    // Phi(z) + z phi(z)
  } else if constexpr (ACT == ACT_GELU_TANH) {                          // z s(v), v = 2 k0 (z + k1 z^3)
    const float z2 = z * z, v = 2.f * GELU_K0 * z * fmaf(GELU_K1, z2, 1.f);
    const float e = fast_exp2(-LOG2E * v), s = fast_rcp(1.f + e);
    return fmaf(z * s * (e * s), 2.f * GELU_K0 * fmaf(3.f * GELU_K1, z2, 1.f), s);
  } else {                                                              // silu
    const float e = fast_exp2(-LOG2E * z), s = fast_rcp(1.f + e);
    return s * fmaf(z, e * s, 1.f);
  }
}

// ---------------------------------------------------------------- splitting the contraction
// A product of few output tiles and a long contraction (the weight gradient: a sum over all tokens; a handful of
// tokens through a wide layer) leaves most SMs without a tile. Its fp32 partial sums then go to slabs of a workspace
// and a second kernel adds them up, always in the same order: no atomics, the same bits every time.
//
// tiles = whole + rest. The first `whole` (a multiple of the units) are walked as they are. Of the others every tile's
// k-blocks are cut into `chunks` of `len`, and each of the rest * chunks pieces has a unit that does its first `head`
// blocks; the units left over share the tails, in order, so that all finish together. Units beside one another work on
// the same k-blocks of different tiles at the same time and share their operands in L2 (cut into one contiguous range
// of (tile, k-block) per unit instead, no two read the same and each tile's operands come from HBM).
struct DensePlan {
  int tiles, units, num_kb;
  int whole, rest, chunks, len, head, tail;   // tail = len - head
  __host__ __device__ int pieces() const { return rest * chunks; }
  __host__ __device__ int helpers() const { return units - pieces(); }
  __host__ __device__ int slots() const { return whole + pieces() + (tail > 0 ? pieces() + helpers() : 0); }
  // helper that does tail block x (helper j has the blocks [j * total / helpers, (j + 1) * total / helpers))
  __host__ __device__ int helper_of(long long x) const {
    const long long total = static_cast<long long>(pieces()) * tail;
    return static_cast<int>(((x + 1) * helpers() - 1) / total);
  }
};

inline DensePlan dense_plan(int tiles, int units, int num_kb, int min_len) {
  DensePlan s{};
  s.tiles = tiles;
  s.units = units;
  s.num_kb = num_kb;
  s.whole = tiles / units * units;
  s.rest = tiles - s.whole;
  if (s.rest == 0) return s;
  int chunks = units / s.rest;
  const int most = num_kb / min_len;
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  s.len = (num_kb + chunks - 1) / chunks;
  s.chunks = (num_kb + s.len - 1) / s.len;
  const int pieces = s.pieces();
  s.head = s.len;
  if (pieces < units && num_kb >= 2 * min_len) {
    const int head = static_cast<int>((static_cast<long long>(s.len) * pieces + units - 1) / units);
    // (worth it where heads and tails are a few blocks long; otherwise the units left over stay idle. Every helper
    // has a block at least: dense_finish_kernel adds up the slabs of all helpers between a tail's first and last)
    if (head >= min_len && s.len - head >= min_len &&
        static_cast<long long>(pieces) * (s.len - head) >= units - pieces)
      s.head = head;
  }
  s.tail = s.len - s.head;
  return s;
}

struct DenseSegment { int tile, kb0, kb1, slot; };

// The segments of one unit, in order.
struct DenseWalk {
  int t;
  long long x, x1;
  bool started;
  __device__ __forceinline__ explicit DenseWalk(int unit) : t(unit), x(0), x1(0), started(false) {}
  __device__ __forceinline__ bool next(const DensePlan& s, int unit, DenseSegment& g) {
    if (t < s.whole) {
      g = {t, 0, s.num_kb, t};
      t += s.units;
      return true;
    }
    const int pieces = s.pieces();
    if (!started) {
      started = true;
      if (unit < pieces) {
        const int c = unit / s.rest;
        g = {s.whole + unit - c * s.rest, c * s.len, c * s.len + s.head, s.whole + unit};
        return true;
      }
      if (s.tail > 0) {
        const long long total = static_cast<long long>(pieces) * s.tail, j = unit - pieces, h = s.helpers();
        x = j * total / h;
        x1 = (j + 1) * total / h;
      }
    }
    if (x >= x1) return false;
    const int v = static_cast<int>(x / s.tail), c = v / s.rest;
    const int off = static_cast<int>(x - static_cast<long long>(v) * s.tail);
    const int n = static_cast<int>(x1 - x < s.tail - off ? x1 - x : s.tail - off);
    const int kb = c * s.len + s.head + off;
    g = {s.whole + v - c * s.rest, kb, kb + n, s.whole + pieces + v + (unit - pieces)};
    x += n;
    return true;
  }
};

}  // namespace strata
