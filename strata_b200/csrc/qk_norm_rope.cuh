// Norm and rotation of query and key heads in one pass, and its gradients.
//
//   r = (mean x^2 + eps)^-1/2,  n = x r,  y = R(p) (n w)        x: one head of one token, w: [head_dim] or none
//   g = R(p)^T dy,  h = g w,    dx = r (h - n mean(h n)),  dw = sum over tokens and heads of g n
//
// R turns `rot` of a head's channels, in pairs of neighbours (2i, 2i + 1) or of the two halves (i, i + rot / 2), by the
// (cos, sin) pairs of the token's table row. Both directions are bound by HBM: a head is read once (twice backward: x
// and dy) and written once, in 16 bits; all arithmetic is fp32.
//
// A group of G lanes (a power of two, 8 channels each) has a head; a warp has a token, S = 32 / G heads of it at a time
// (several tokens where both q and k have fewer heads than that), in steps of two rounds of q heads or of k heads. So
// the token's table row is read and unpacked once for all its heads. A head whose width is no power of two leaves the
// group's last lanes idle. What a step reads is asked for two steps ahead with cp.async into slots of shared memory
// that only the asking lane reads (but for shared table rows): bytes in flight that cost no registers, and no barrier.
// Divisions by launch constants are multiplications; arithmetic runs on fp32 pairs.
// Measured (8 + 8 heads of 64, 262144 tokens, bf16, half table; the bytes alone take 166 us forward, 250 backward):
// forward 198 us, backward 292 (178 and 263 without rotation). With the loads straight into registers, two rounds of q
// and two of k at a time: 190 and 355 (16 + 4 heads of 128: 303 against 248, 370 against 323); more blocks per SM at
// fewer registers spill (backward, three blocks: 353).
#pragma once
#include "dense_common.cuh"

namespace strata {

constexpr int QK_ROUNDS = 2;          // rounds of q heads, and of k heads, in flight

struct QkTensor {                     // [tokens, heads, head_dim], unit channel stride, 16-byte pieces
  const void* p;
  long long token, head;              // strides in elements
};
// Division by a number that the host knows: n / d = (n mul) >> 32 >> shift for n < 2^31 (Granlund and Montgomery 1994).
struct QkDiv {
  uint32_t d, mul, shift;
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};
inline QkDiv qk_div(uint32_t d) {      // 2^31 > d >= 1
  QkDiv q{d, 0, 0};
  if (d <= 1) return q;
  while ((1ull << (q.shift + 1)) < d) ++q.shift;            // 2^shift < d <= 2^(shift + 1)
  q.mul = static_cast<uint32_t>(((1ull << (32 + q.shift)) + d - 1) / d);
  return q;
}

struct QkParams {
  QkTensor x[2];                      // q, k
  QkTensor y[2];                      // outputs (of the backward pass: dx)
  QkTensor dy[2];                     // backward
  const float* w[2];                  // [head_dim] or nullptr
  int heads[2];
  int part[2];                        // heads of a block: block (x, y) has those from y part on
  int head_dim, rot;
  const void* table;                  // [rows, rot / 2] (cos, sin) pairs, half or float; nullptr: no rotation
  int table_f32, table_rows;
  const void* positions;              // [M] int32 or int64, or nullptr: row m / tokens_per_tile * hw + m % hw
  int positions_64;
  QkDiv tokens_per_tile, hw;
  long long M;
  float eps;
  float* partial;                     // backward: [grid, 2, head_dim] sums of dw, or nullptr
};

enum QkTable : int { QK_NO_TABLE = 0, QK_HALF_TABLE = 1, QK_F32_TABLE = 2 };
// How a token's heads come: QK_ROUNDS rounds of q heads or of k heads a step; the same for a part of them, the other
// parts in other blocks; a round of q heads and one of k heads a step, which are all.
enum QkHeads : int { QK_ALL = 0, QK_PARTS = 1, QK_FEW = 2 };

// Table row of token m; -1: a padding token, -2: no such row.
__device__ __forceinline__ int qk_row(const QkParams& p, long long m) {
  if (p.positions == nullptr) {
    const unsigned t = static_cast<unsigned>(m);
    return static_cast<int>(p.tokens_per_tile.div(t) * p.hw.d + t - p.hw.div(t) * p.hw.d);
  }
  const long long r = p.positions_64 ? __ldg(static_cast<const long long*>(p.positions) + m)
                                     : __ldg(static_cast<const int*>(p.positions) + m);
  if (r >= p.table_rows) return -2;
  return r < 0 ? -1 : static_cast<int>(r);
}

// (cos, sin) for this lane's channels 8 v .. 8 v + 7: four pairs where neighbours turn, else one for each channel; (1,
// 0) where nothing turns. sin has the sign with which a pair's second channel enters its first: -1 forward, +1 for the
// inverse turn; for channels of the second half the other sign.
// raw: the lane's part of the table row, TV 16-byte vectors.
template <int TAB, bool ADJ>
struct QkTab {
  static constexpr int N = ADJ ? 4 : 8;
  static constexpr int TV = TAB == QK_NO_TABLE ? 0 : (TAB == QK_F32_TABLE ? 2 : 1) * (ADJ ? 1 : 2);
};
// First table entry of this lane in a row of rot / 2.
template <bool ADJ>
__device__ __forceinline__ int qk_entry(const QkParams& p, int v) {
  const int half = p.rot >> 1;
  return ADJ ? 4 * v : 8 * v >= half ? 8 * v - half : 8 * v;
}
template <int TAB, bool ADJ, int N, int TV>
__device__ __forceinline__ void qk_table(const QkParams& p, const uint4 (&raw)[TV], bool turns, int v, float sign,
                                         float (&c)[N], float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < TV; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (TAB == QK_F32_TABLE) {
        if (k & 1) s[2 * i + k / 2] = __uint_as_float(w[k]); else c[2 * i + k / 2] = __uint_as_float(w[k]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        c[4 * i + k] = f.x; s[4 * i + k] = f.y;
      }
    }
  }
  if (!ADJ && 8 * v >= p.rot >> 1) sign = -sign;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c[i] = turns ? c[i] : 1.f;
    s[i] = turns ? sign * s[i] : 0.f;
  }
}

// A lane's eight channels as four fp32 pairs. Where neighbours turn the pairs are (0, 2), (4, 6), (1, 3), (5, 7), so
// that the rotation multiplies whole pairs: even' = even c + odd s, odd' = odd c - even s; else (0, 1), (2, 3), ...
template <bool ADJ>
__device__ constexpr int qk_first(int i) { return ADJ ? (i & 1) * 4 + (i >> 1) : 2 * i; }
template <bool ADJ>
__device__ constexpr int qk_second(int i) { return qk_first<ADJ>(i) + (ADJ ? 2 : 1); }

template <typename T, bool ADJ>
__device__ __forceinline__ void qk_unpack(const uint4& u, uint64_t (&x)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  auto at = [&](int ch) { return ch & 1 ? Pair16<T>::hi(w[ch >> 1]) : Pair16<T>::lo(w[ch >> 1]); };
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2(at(qk_first<ADJ>(i)), at(qk_second<ADJ>(i)));
}
template <typename T, bool ADJ>
__device__ __forceinline__ uint4 qk_pack(const uint64_t (&x)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(x[i], f[qk_first<ADJ>(i)], f[qk_second<ADJ>(i)]);
  return make_uint4(Pair16<T>::pack(f[0], f[1]), Pair16<T>::pack(f[2], f[3]), Pair16<T>::pack(f[4], f[5]),
                    Pair16<T>::pack(f[6], f[7]));
}

// Turns a lane's channels. partner: the lane that has their partners (halves; all lanes of the warp take part).
template <bool ADJ, int N>
__device__ __forceinline__ void qk_turn(const float (&c)[N], const float (&s)[N], int partner, uint64_t (&x)[4]) {
  if constexpr (ADJ) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {      // pairs (0, 2) with (1, 3), (4, 6) with (5, 7)
      const uint64_t c2 = pack2(c[2 * i], c[2 * i + 1]), s2 = pack2(s[2 * i], s[2 * i + 1]),
                     n2 = pack2(-s[2 * i], -s[2 * i + 1]);
      const uint64_t e = x[i], o = x[i + 2];
      x[i] = ffma2(o, s2, fmul2(e, c2));
      x[i + 2] = ffma2(e, n2, fmul2(o, c2));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      unpack2(x[i], a, b);
      a = __shfl_sync(0xffffffffu, a, partner);
      b = __shfl_sync(0xffffffffu, b, partner);
      x[i] = ffma2(pack2(a, b), pack2(s[2 * i], s[2 * i + 1]), fmul2(x[i], pack2(c[2 * i], c[2 * i + 1])));
    }
  }
}

__device__ __forceinline__ float qk_dot(const uint64_t (&a)[4], const uint64_t (&b)[4]) {
  uint64_t t = fmul2(a[0], b[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) t = ffma2(a[i], b[i], t);
  float lo, hi;
  unpack2(t, lo, hi);
  return lo + hi;
}
template <int G>
__device__ __forceinline__ float qk_group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One head's vector of this lane: y of x, or dx of x and dy = gr and its part of dw (if it counts: a head that exists,
// of a token that is not padding).
template <typename T, int G, int TAB, bool ADJ, bool GRAD, int N>
__device__ __forceinline__ uint4 qk_vector(const uint4& xr, const uint4& gr, const float (&w)[8], const float (&c)[N],
                                           const float (&s)[N], int partner, bool counts, float inv, float eps,
                                           uint64_t (&sums)[4]) {
  uint64_t x[4], h[4];
  qk_unpack<T, ADJ>(xr, x);
  auto weighted = [&](uint64_t v, int i) {
    float a, b;
    unpack2(v, a, b);
    return pack2(a * w[qk_first<ADJ>(i)], b * w[qk_second<ADJ>(i)]);
  };
  float sq = qk_dot(x, x);
  if constexpr (!GRAD) {
    const float rs = rsqrtf(fmaf(qk_group_sum<G>(sq), inv, eps));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = weighted(x[i], i);
    if constexpr (TAB != QK_NO_TABLE) qk_turn<ADJ>(c, s, partner, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = fmul2(h[i], pack2(rs, rs));
    return qk_pack<T, ADJ>(h);
  } else {
    uint64_t g[4];
    qk_unpack<T, ADJ>(gr, g);
    if constexpr (TAB != QK_NO_TABLE) qk_turn<ADJ>(c, s, partner, g);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = weighted(g[i], i);
    float dot = qk_dot(h, x);
#pragma unroll
    for (int ofs = G / 2; ofs > 0; ofs >>= 1) {
      sq += __shfl_xor_sync(0xffffffffu, sq, ofs);
      dot += __shfl_xor_sync(0xffffffffu, dot, ofs);
    }
    // dx = r (h - x r^2 mean(h x)), h = g w;  dw += g (x r). (r^3 by itself leaves fp32 at an rms of 1e13 or 1e-13)
    const float rs = rsqrtf(fmaf(sq, inv, eps)), b = -(rs * (dot * inv)) * rs;
    const uint64_t r2 = pack2(rs, rs), b2 = pack2(b, b);
    if (counts) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[i] = ffma2(g[i], fmul2(x[i], r2), sums[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = fmul2(ffma2(x[i], b2, h[i]), r2);
    return qk_pack<T, ADJ>(h);
  }
}

// Weights of this lane's channels. (Read again for every token, from L1: registers that the loop does not have to
// keep.)
__device__ __forceinline__ void qk_weights(const float* w, int v, float (&o)[8]) {
  if (w != nullptr) {
    const float4* f = reinterpret_cast<const float4*>(w) + 2 * v;
    const float4 a = __ldg(f), b = __ldg(f + 1);
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 1.f;
  }
}

// Bytes a lane asks for ahead, past the registers: into its own 16-byte slots of shared memory (zeros where on is
// false).
__device__ __forceinline__ void qk_ask(uint32_t slot, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 qk_got(uint32_t slot) {
  uint4 u;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(slot) : "memory");
  return u;
}

// A stage of a warp: the lanes' vectors, the table's, and the lanes' table rows. The table's vectors are each lane's
// own like the others, or (SHARE) those of the tokens' rows side by side, each loaded once by whichever lane and read
// by all that need it: where a lane needs four, 64 bytes from the next lane's, and two beside a single step's vectors.
// Own / shared, microseconds forward, 142667 tokens of 4 + 4 heads of 64: four 188 / 93, two 87 / 79, one 60 / 64;
// 65536 of 16 + 4 heads of 128: four 169 / 164, two 145 / 152; 262144 of 8 + 8 heads of 64, one: 200 / 219.
template <int TAB, bool ADJ, bool GRAD, int HEADS>
struct QkRing {
  static constexpr int STAGES = 3;
  static constexpr int TV = QkTab<TAB, ADJ>::TV;
  static constexpr bool SHARE = TV == 4 || (TV == 2 && HEADS == QK_FEW);
  static constexpr int VECTORS = (GRAD ? 2 : 1) * QK_ROUNDS;                      // of a lane
  static constexpr int TABLE = SHARE ? (TAB == QK_F32_TABLE ? 2 : 1) : TV;
  static constexpr int ROWS = (VECTORS + TABLE) * 512;
  static constexpr int STAGE = ROWS + (TAB == QK_NO_TABLE ? 0 : 128);
  static constexpr int BYTES = 8 * STAGES * STAGE;
};

// GRAD false: y; true: dx and the sums of dw. Blocks of 256 threads, a stride loop over the tokens, steps asked for
// STAGES - 1 ahead. Kernels of their own for the ways of the heads: with the limits of QK_PARTS in registers the loop
// over many tokens is 5 to 11 % slower; QK_FEW has twice the bytes in flight of two half-empty steps (64458 tokens of
// 4 + 4 heads of 64: 46 us -> 35, backward 64 -> 48).
template <typename T, int G, int TAB, bool ADJ, bool GRAD, int HEADS>
__global__ void __launch_bounds__(256, GRAD ? 2 : 4) qk_norm_rope_kernel(const QkParams p) {
  using Ring = QkRing<TAB, ADJ, GRAD, HEADS>;
  constexpr bool SPLIT = HEADS == QK_PARTS, FEW = HEADS == QK_FEW;
  constexpr int S = 32 / G, R = QK_ROUNDS, N = QkTab<TAB, ADJ>::N, TV = QkTab<TAB, ADJ>::TV, D = Ring::STAGES;
  extern __shared__ uint4 ring[];
  chain_begin();
  const int lane = threadIdx.x & 31, sub = lane / G, v_raw = lane & (G - 1);
  const bool lane_on = 8 * v_raw < p.head_dim, turns = 8 * v_raw < p.rot;
  const int v = lane_on ? v_raw : 0;
  const int hv = p.rot >> 4;                       // vectors in half the turned channels
  const int partner = ADJ ? lane : v_raw < hv ? lane + hv : v_raw < 2 * hv ? lane - hv : lane;
  const float inv = 1.0f / static_cast<float>(p.head_dim);
  const uint32_t slots = smem_u32(ring) + (threadIdx.x >> 5) * (D * Ring::STAGE) + lane * 16;
  const uint32_t rows = slots + Ring::ROWS - lane * 12;
  // heads side by side in the warp, and the tokens that leaves room for
  int width = 1;
  while (width < S && (width < p.part[0] || width < p.part[1])) width *= 2;
  const int tokens = S / width, head = sub & (width - 1), tok = sub / width;
  // the block's heads: lim of them from base on (none: lim <= 0)
  const int part = SPLIT ? blockIdx.y : 0;
  const int lim_q = SPLIT ? min(p.heads[0] - part * p.part[0], p.part[0]) : 0;
  const int lim_k = SPLIT ? min(p.heads[1] - part * p.part[1], p.part[1]) : 0;
  auto base = [&](int k) { return SPLIT ? part * p.part[k] : 0; };
  auto lim = [&](int k) { return !SPLIT ? p.heads[k] : k == 0 ? lim_q : lim_k; };
  const uint32_t M = static_cast<uint32_t>(p.M), stride = gridDim.x * (blockDim.x >> 5) * tokens;
  const uint32_t first = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * tokens;
  auto at = [&](const QkTensor& t, uint32_t m, int h) {
    return const_cast<uint16_t*>(static_cast<const uint16_t*>(t.p)) + static_cast<long long>(m) * t.token +
           static_cast<long long>(h) * t.head + 8 * v;
  };
  // SHARE: lane j asks for vector j (fp32: and j + 32) of the tokens' table rows; swizzled, so that eight lanes'
  // vectors are in different banks
  constexpr int PER = TAB == QK_F32_TABLE ? 2 : 4;          // entries of a vector
  const uint32_t tab0 = slots - lane * 16 + Ring::VECTORS * 512;
  auto tab_at = [](int x) { return static_cast<uint32_t>(x ^ ((x >> 3) & 3)) * 16u; };
  [[maybe_unused]] int row_vectors = 1, tab_token[2] = {0, 0}, tab_vector[2] = {0, 0}, tab_first = 0;
  if constexpr (Ring::SHARE) {
    row_vectors = (p.rot >> 1) / PER;
#pragma unroll
    for (int q = 0; q < Ring::TABLE; ++q) {
      tab_token[q] = (lane + 32 * q) / row_vectors;
      tab_vector[q] = lane + 32 * q - tab_token[q] * row_vectors;
    }
    tab_first = tok * row_vectors + (turns ? qk_entry<ADJ>(p, v_raw) / PER : 0);
  }
  // the step that is asked for next: token m_a (of the warp's first lanes), tensor k_a, heads from h_a; its stage
  uint32_t m_a = first;
  int k_a = 0, h_a = 0, stage_a = 0, row_a = 0;
  if (TAB != QK_NO_TABLE && first + tok < M) row_a = qk_row(p, first + tok);
  auto ask = [&]() {
    if (m_a < M) {
      const uint32_t slot = slots + stage_a * Ring::STAGE, m = m_a + tok;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int k = FEW ? r : k_a, h = FEW ? head : h_a + r * width + head;
        const bool on = lane_on && m < M && h < lim(k);
        qk_ask(slot + r * 512, at(p.x[k], on ? m : 0, on ? base(k) + h : 0), on);
        if constexpr (GRAD) qk_ask(slot + (R + r) * 512, at(p.dy[k], on ? m : 0, on ? base(k) + h : 0), on);
      }
      if (TAB != QK_NO_TABLE && (FEW || (k_a == 0 && h_a == 0))) {
        if (m >= M) row_a = -1;
        const char* table = static_cast<const char*>(p.table);
        if constexpr (Ring::SHARE) {
#pragma unroll
          for (int q = 0; q < Ring::TABLE; ++q) {
            const int row = __shfl_sync(0xffffffffu, row_a, tab_token[q] * (width * G) & 31);
            const bool there = tab_token[q] < tokens, on = there && row >= 0;
            const long long at16 = on ? static_cast<long long>(row) * row_vectors + tab_vector[q] : 0;
            if (there) qk_ask(tab0 + stage_a * Ring::STAGE + tab_at(lane + 32 * q), table + at16 * 16, on);
          }
        } else {
          const bool on = turns && row_a >= 0;
          const long long e =
              (on ? static_cast<long long>(row_a) * (p.rot >> 1) : 0) + (turns ? qk_entry<ADJ>(p, v_raw) : 0);
#pragma unroll
          for (int i = 0; i < TV; ++i)
            qk_ask(slot + (Ring::VECTORS + i) * 512, table + e * (16 / PER) + i * 16, on);
        }
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(rows + stage_a * Ring::STAGE), "r"(row_a) : "memory");
        if (m + stride < M) row_a = qk_row(p, m + stride);       // (the next token's, a token ahead)
      }
      if constexpr (FEW) {
        m_a += stride;
      } else if ((h_a += R * width) >= lim(k_a)) {
        h_a = 0;
        if (++k_a == 2) {
          k_a = 0;
          m_a += stride;
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_a = stage_a + 1 == D ? 0 : stage_a + 1;
  };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) ask();
  uint64_t sums[2][4];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[k][i] = 0ull;
  int stage = 0;
  // (m0: the warp's first token, the same for all lanes)
  for (uint32_t m0 = first; m0 < M; m0 += stride) {
    const uint32_t m = m0 + tok;
    int row = 0;
    float c[N], s[N], w[8];
    auto arrive = [&](bool with_table) {      // the next step's slot
      if constexpr (Ring::SHARE) __syncwarp();        // (all have read the last step's table rows)
      ask();
      asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
      const uint32_t slot = slots + stage * Ring::STAGE;
      if (TAB != QK_NO_TABLE && with_table) {
        if constexpr (Ring::SHARE) __syncwarp();
        uint4 raw[TV > 0 ? TV : 1];
#pragma unroll
        for (int i = 0; i < TV; ++i)
          raw[i] = qk_got(Ring::SHARE ? tab0 + stage * Ring::STAGE + tab_at(tab_first + i)
                                      : slot + (Ring::VECTORS + i) * 512);
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(row) : "r"(rows + stage * Ring::STAGE) : "memory");
        if (row == -2) atomicCAS(&g_status, 0, ST_BAD_POSITION);
        if constexpr (TAB != QK_NO_TABLE)
          qk_table<TAB, ADJ>(p, raw, turns && row >= 0, v_raw, GRAD ? 1.f : -1.f, c, s);
      }
      stage = stage + 1 == D ? 0 : stage + 1;
      return slot;
    };
    auto round = [&](uint32_t slot, int r, int k, int h) {
      const uint4 xr = qk_got(slot + r * 512), gr = GRAD ? qk_got(slot + (R + r) * 512) : xr;
      // (a slot without a head holds zeros, whose 1 / r has no bound but eps: 0 times infinity where that is 0)
      const bool counts = GRAD && lane_on && m < M && h < lim(k) && (TAB == QK_NO_TABLE || row >= 0);
      uint4 o = qk_vector<T, G, TAB, ADJ, GRAD>(xr, gr, w, c, s, partner, counts, inv, p.eps, sums[k]);
      if (TAB != QK_NO_TABLE && p.positions != nullptr && row < 0) {     // padding: zero; behind the table: NaN
        const uint32_t u = row == -1 ? 0u : 0x7FFF7FFFu;
        o = make_uint4(u, u, u, u);
      }
      if (lane_on && m < M && h < lim(k)) *reinterpret_cast<uint4*>(at(p.y[k], m, base(k) + h)) = o;
    };
    if constexpr (FEW) {
      static_assert(R == 2, "q and k");
      const uint32_t slot = arrive(true);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        qk_weights(p.w[k], v, w);
        round(slot, k, k, head);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {      // (a part without k heads: an empty step)
        for (int h0 = 0; (SPLIT && h0 == 0) || h0 < lim(k); h0 += R * width) {
          const uint32_t slot = arrive(k == 0 && h0 == 0);
          qk_weights(p.w[k], v, w);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (r > 0 && h0 + r * width >= lim(k)) continue;       // (the same for the block)
            round(slot, r, k, h0 + r * width + head);
          }
        }
      }
    }
  }
  if constexpr (GRAD) {
    if (p.partial == nullptr) return;
    // (the ring is empty: steps past the last token were not asked for)
    float* red = reinterpret_cast<float*>(ring);       // [8][2][G * 8]
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float t[2];
        unpack2(sums[k][i], t[0], t[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = G; o < 32; o <<= 1) t[e] += __shfl_xor_sync(0xffffffffu, t[e], o);
          if (sub == 0)
            red[((threadIdx.x >> 5) * 2 + k) * (G * 8) + 8 * v_raw + (e ? qk_second<ADJ>(i) : qk_first<ADJ>(i))] = t[e];
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += 256) {
      const int k = i >= p.head_dim ? 1 : 0, ch = i - k * p.head_dim;
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += red[(w * 2 + k) * (G * 8) + ch];
      p.partial[(static_cast<long long>(part) * gridDim.x + blockIdx.x) * 2 * p.head_dim + i] = t;
    }
  }
}

// dw: the blocks' sums in their order. Eight channels a block, 32 rows of sums side by side.
__global__ void __launch_bounds__(256) qk_weight_grad_kernel(const float* partial, int rows, int head_dim, float* dq,
                                                             float* dk) {
  chain_begin();
  __shared__ float red[32][9];
  const int col = blockIdx.x * 8 + (threadIdx.x & 7), r0 = threadIdx.x >> 3;
  float a = 0.f;
#pragma unroll 8
  for (int r = r0; r < rows; r += 32) a += partial[static_cast<long long>(r) * 2 * head_dim + col];
  red[r0][threadIdx.x & 7] = a;
  __syncthreads();
  if (r0 != 0) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) a += red[i][threadIdx.x & 7];
  if (col < head_dim) {
    if (dq) dq[col] = a;
  } else if (dk) {
    dk[col - head_dim] = a;
  }
}

inline int qk_group(int head_dim) {      // (16 channels in two lanes are no narrower than 32 in four)
  int g = 4;
  while (g * 8 < head_dim) g *= 2;
  return g;
}
// A token a warp: no more blocks than that takes, and no more than run at once backward (a row of sums each).
inline long long qk_most_blocks(bool grad, int sms) { return static_cast<long long>(sms) * (grad ? 2 : 16); }
// Grid for p's tokens and heads; sets p.part. Where the tokens leave room for that, a token's heads go to several
// blocks, down to one round of q heads each (44 tokens, 48 + 12 heads of 256, in a row of calls: forward 29.3 us ->
// 13.0, backward 38.7 -> 16.7; from 300 tokens of 12 + 12 heads of 64 on no difference).
inline dim3 qk_grid(QkParams& p, bool grad, int sms) {
  const long long blocks = (p.M + 7) / 8, cap = qk_most_blocks(grad, sms);
  p.part[0] = p.heads[0];
  p.part[1] = p.heads[1];
  const int side = 32 / qk_group(p.head_dim);
  long long parts = 2LL * sms / blocks;
  if (parts > (p.heads[0] + side - 1) / side) parts = (p.heads[0] + side - 1) / side;
  if (parts > 1) {
    p.part[0] = static_cast<int>((p.heads[0] + parts - 1) / parts);
    parts = (p.heads[0] + p.part[0] - 1) / p.part[0];
    p.part[1] = static_cast<int>((p.heads[1] + parts - 1) / parts);
  } else {
    parts = 1;
  }
  return dim3(static_cast<unsigned>(blocks < cap ? blocks : cap), static_cast<unsigned>(parts));
}

template <typename T, int G, int TAB, bool ADJ, bool GRAD, int HEADS>
inline int launch_qk_s(const QkParams& p, dim3 grid, cudaStream_t st) {
  auto kern = qk_norm_rope_kernel<T, G, TAB, ADJ, GRAD, HEADS>;
  constexpr int bytes = QkRing<TAB, ADJ, GRAD, HEADS>::BYTES;
  static_assert(bytes >= 8 * 2 * G * 8 * 4, "the sums of a block");
  static std::atomic<uint64_t> smem_set;
  if (const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), bytes, smem_set); e != cudaSuccess)
    return -static_cast<int>(e) - 1000;
  return launch_chained(kern, grid, 256, bytes, st, 1, p);
}
template <typename T, int G, int TAB, bool ADJ, bool GRAD>
inline int launch_qk_k(const QkParams& p, dim3 grid, cudaStream_t st) {
  if (grid.y > 1) return launch_qk_s<T, G, TAB, ADJ, GRAD, QK_PARTS>(p, grid, st);
  return p.heads[0] <= 32 / G && p.heads[1] <= 32 / G ? launch_qk_s<T, G, TAB, ADJ, GRAD, QK_FEW>(p, grid, st)
                                                      : launch_qk_s<T, G, TAB, ADJ, GRAD, QK_ALL>(p, grid, st);
}
template <typename T, int G, bool GRAD>
inline int launch_qk_t(const QkParams& p, bool adjacent, dim3 grid, cudaStream_t st) {
  if (p.table == nullptr) return launch_qk_k<T, G, QK_NO_TABLE, true, GRAD>(p, grid, st);
  if (p.table_f32)
    return adjacent ? launch_qk_k<T, G, QK_F32_TABLE, true, GRAD>(p, grid, st)
                    : launch_qk_k<T, G, QK_F32_TABLE, false, GRAD>(p, grid, st);
  return adjacent ? launch_qk_k<T, G, QK_HALF_TABLE, true, GRAD>(p, grid, st)
                  : launch_qk_k<T, G, QK_HALF_TABLE, false, GRAD>(p, grid, st);
}
template <typename T, bool GRAD>
inline int launch_qk_g(const QkParams& p, bool adjacent, dim3 grid, cudaStream_t st) {
  switch (qk_group(p.head_dim)) {
    case 4: return launch_qk_t<T, 4, GRAD>(p, adjacent, grid, st);
    case 8: return launch_qk_t<T, 8, GRAD>(p, adjacent, grid, st);
    case 16: return launch_qk_t<T, 16, GRAD>(p, adjacent, grid, st);
    default: return launch_qk_t<T, 32, GRAD>(p, adjacent, grid, st);
  }
}
template <bool GRAD>
inline int launch_qk(const QkParams& p, bool adjacent, bool fp16, dim3 grid, cudaStream_t st) {
  return fp16 ? launch_qk_g<__half, GRAD>(p, adjacent, grid, st)
              : launch_qk_g<__nv_bfloat16, GRAD>(p, adjacent, grid, st);
}

}  // namespace strata
