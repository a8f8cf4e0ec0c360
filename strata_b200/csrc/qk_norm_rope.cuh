// Norm and rotation of query and key heads in one pass, and its gradients.
//
//   r = (mean x^2 + eps)^-1/2,  n = x r,  y = R(p) (n w)        x: one head of one token, w: [head_dim] or none
//   g = R(p)^T dy,  h = g w,    dx = r (h - n mean(h n)),  dw = sum over tokens and heads of g n
//
// R turns `rot` of a head's channels, in pairs of neighbours (2i, 2i + 1) or of the two halves (i, i + rot / 2), by the
// (cos, sin) pairs of the token's table row. Both directions are bound by HBM: a head is read once (twice backward: x
// and dy) and written once, in 16 bits; all arithmetic is fp32.
//
// A group of G lanes (a power of two, 8 channels each) has a head, a warp 32 / G heads at a time; an item of work is
// one token's next U rounds of heads, whose loads are all in flight together. The table row is read once per item
// and not per head: the lanes of a group need the same channels of every head. A head whose width is no power of two
// leaves the group's last lanes idle. Pairs of the two halves meet through a shuffle within the group.
#pragma once
#include "dense_common.cuh"

namespace strata {

constexpr int QK_ROUNDS = 4;          // U

struct QkTensor {                     // [tokens, heads, head_dim], unit channel stride, 16-byte pieces
  const void* p;
  long long token, head;              // strides in elements
};
struct QkParams {
  QkTensor x[2];                      // q, k
  QkTensor y[2];                      // outputs (of the backward pass: dx)
  QkTensor dy[2];                     // backward
  const float* w[2];                  // [head_dim] or nullptr
  int heads[2];
  int head_dim, rot;
  const void* table;                  // [rows, rot / 2] (cos, sin) pairs, half or float; nullptr: no rotation
  int table_f32, table_rows;
  const void* positions;              // [M] int32 or int64, or nullptr: row m / tokens_per_tile * hw + m % hw
  int positions_64;
  int tokens_per_tile, hw;
  long long M;
  float eps;
  float* partial;                     // backward: [grid, 2, head_dim] sums of dw, or nullptr
};

// Table row of token m; -1: a padding token, -2: no such row.
__device__ __forceinline__ int qk_row(const QkParams& p, long long m) {
  if (p.table == nullptr) return 0;
  if (p.positions == nullptr) return static_cast<int>(m / p.tokens_per_tile * p.hw + m % p.hw);
  const long long r = p.positions_64 ? __ldg(static_cast<const long long*>(p.positions) + m)
                                     : __ldg(static_cast<const int*>(p.positions) + m);
  if (r >= p.table_rows) return -2;
  return r < 0 ? -1 : static_cast<int>(r);
}

// The (cos, sin) of this lane's channels 8 v .. 8 v + 7: of four neighbour pairs, or of eight pairs of the two halves
// (the same ones for both partners). One of c, s for each channel; c = 1, s = 0 where nothing turns. Neighbours: s has
// the sign with which the partner enters (-sin for the even channel), so that y_i = x_i c_i + x_partner s_i.
template <bool ADJ>
__device__ __forceinline__ void qk_table(const QkParams& p, int row, int v, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = 1.f; s[i] = 0.f; }
  if (p.table == nullptr || row < 0 || 8 * v >= p.rot) return;
  const int half = p.rot >> 1;
  const int pair0 = ADJ ? 4 * v : (8 * v < half ? 8 * v : 8 * v - half);
  constexpr int N = ADJ ? 4 : 8;
  float cc[N], ss[N];
  const long long at = static_cast<long long>(row) * half + pair0;
  if (p.table_f32) {
    const float4* t = reinterpret_cast<const float4*>(static_cast<const float2*>(p.table) + at);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float4 f = __ldg(t + i);
      cc[2 * i] = f.x; ss[2 * i] = f.y; cc[2 * i + 1] = f.z; ss[2 * i + 1] = f.w;
    }
  } else {
    const uint4* t = reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(p.table) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 u = __ldg(t + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        cc[4 * i + k] = f.x; ss[4 * i + k] = f.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (ADJ) {
      c[i] = cc[i >> 1];
      s[i] = i & 1 ? ss[i >> 1] : -ss[i >> 1];
    } else {
      c[i] = cc[i];
      s[i] = 8 * v < half ? -ss[i] : ss[i];
    }
  }
}

// x <- x c + partner s, in the group (all lanes of the warp take part in the shuffles). sign -1: the inverse turn.
template <bool ADJ>
__device__ __forceinline__ void qk_turn(const QkParams& p, int v, const float (&c)[8], const float (&s)[8], float sign,
                                        float (&x)[8]) {
  float o[8];
  if constexpr (ADJ) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = x[i ^ 1];
  } else {
    const int hv = p.rot >> 4;                             // vectors in half the turned channels
    const int lane = threadIdx.x & 31;
    const int from = v < hv ? lane + hv : v < 2 * hv ? lane - hv : lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, x[i], from);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], c[i], sign * s[i] * o[i]);
}

template <typename T>
__device__ __forceinline__ void qk_unpack(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Pair16<T>::lo(w[i]);
    x[2 * i + 1] = Pair16<T>::hi(w[i]);
  }
}
template <typename T>
__device__ __forceinline__ uint4 qk_pack(const float (&x)[8]) {
  return make_uint4(Pair16<T>::pack(x[0], x[1]), Pair16<T>::pack(x[2], x[3]), Pair16<T>::pack(x[4], x[5]),
                    Pair16<T>::pack(x[6], x[7]));
}
template <int G>
__device__ __forceinline__ float qk_group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint4 qk_load(const QkTensor& t, long long m, int head, int v) {
  // (a plain load: y may be x)
  return reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t.p) + m * t.token + head * t.head)[v];
}
__device__ __forceinline__ void qk_store(const QkTensor& t, long long m, int head, int v, const uint4& u) {
  reinterpret_cast<uint4*>(const_cast<uint16_t*>(static_cast<const uint16_t*>(t.p)) + m * t.token + head * t.head)[v] = u;
}
__device__ __forceinline__ void qk_weights(const float* w, int v, bool live, float (&o)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = w != nullptr && live ? __ldg(w + 8 * v + i) : 1.f;
}

// GRAD false: y; true: dx and the sums of dw. Blocks of 256 threads, a stride loop over the items.
template <typename T, int G, bool ADJ, bool GRAD>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkParams p) {
  constexpr int S = 32 / G, U = QK_ROUNDS;
  chain_begin();
  const int lane = threadIdx.x & 31, v = lane & (G - 1), sub = lane / G;
  const bool live = 8 * v < p.head_dim;
  const int heads = p.heads[0] + p.heads[1], chunks = (heads + S * U - 1) / (S * U);
  const float inv = 1.0f / static_cast<float>(p.head_dim);
  float wq[8], wk[8];
  qk_weights(p.w[0], v, live, wq);
  qk_weights(p.w[1], v, live, wk);
  [[maybe_unused]] float sums[2][8];
  if constexpr (GRAD) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[0][i] = sums[1][i] = 0.f;
  }
  const long long items = p.M * chunks;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long it = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items;
       it += warps) {
    const long long m = it / chunks;
    const int h0 = static_cast<int>(it - m * chunks) * (S * U) + sub;
    uint4 xr[U], gr[GRAD ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * S;
      const bool on = live && h < heads;
      const int k = h >= p.heads[0] ? 1 : 0, hh = h - (k ? p.heads[0] : 0);
      xr[u] = on ? qk_load(p.x[k], m, hh, v) : make_uint4(0u, 0u, 0u, 0u);
      if constexpr (GRAD) gr[u] = on ? qk_load(p.dy[k], m, hh, v) : make_uint4(0u, 0u, 0u, 0u);
    }
    const int row = qk_row(p, m);
    float c[8], s[8];
    qk_table<ADJ>(p, row, v, c, s);
    if (row == -2 && lane == 0) atomicCAS(&g_status, 0, ST_BAD_POSITION);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * S;
      const int k = h >= p.heads[0] ? 1 : 0, hh = h - (k ? p.heads[0] : 0);
      float x[8];
      qk_unpack<T>(xr[u], x);
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], sq);
      const float r = rsqrtf(fmaf(qk_group_sum<G>(sq), inv, p.eps));
      float out[8];
      if constexpr (!GRAD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = x[i] * r * (k ? wk[i] : wq[i]);
        if (p.table != nullptr) qk_turn<ADJ>(p, v, c, s, 1.f, out);
      } else {
        float g[8];
        qk_unpack<T>(gr[u], g);
        if (p.table != nullptr) qk_turn<ADJ>(p, v, c, s, -1.f, g);
        if (row < 0) {        // padding, whatever x and dy hold there: no part of dw (a bad position: NaN, below)
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = 0.f;
        }
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = row < 0 ? 0.f : x[i] * r;                    // n
          if (k) sums[1][i] = fmaf(g[i], x[i], sums[1][i]);
          else sums[0][i] = fmaf(g[i], x[i], sums[0][i]);
          g[i] *= k ? wk[i] : wq[i];
          dot = fmaf(g[i], x[i], dot);
        }
        dot = qk_group_sum<G>(dot) * inv;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = r * fmaf(-x[i], dot, g[i]);
      }
      if (live && h < heads) {
        if (row == -1) {
          qk_store(p.y[k], m, hh, v, make_uint4(0u, 0u, 0u, 0u));
        } else {
          if (row < 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) out[i] = __int_as_float(0x7FC00000);
          }
          qk_store(p.y[k], m, hh, v, qk_pack<T>(out));
        }
      }
    }
  }
  if constexpr (GRAD) {
    if (p.partial == nullptr) return;
    __shared__ float red[8][2][G * 8];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float t = sums[k][i];
#pragma unroll
        for (int o = G; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (sub == 0) red[threadIdx.x >> 5][k][8 * v + i] = t;
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += 256) {
      const int k = i >= p.head_dim ? 1 : 0, ch = i - k * p.head_dim;
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += red[w][k][ch];
      p.partial[static_cast<long long>(blockIdx.x) * 2 * p.head_dim + i] = t;
    }
  }
}

// dw: the blocks' sums in their order. 32 channels a block, eight rows of sums side by side.
__global__ void __launch_bounds__(256) qk_weight_grad_kernel(const float* partial, int rows, int head_dim, float* dq,
                                                             float* dk) {
  chain_begin();
  __shared__ float red[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), r0 = threadIdx.x >> 5;
  float a = 0.f;
  if (col < 2 * head_dim) {
#pragma unroll 8
    for (int r = r0; r < rows; r += 8) a += partial[static_cast<long long>(r) * 2 * head_dim + col];
  }
  red[r0][threadIdx.x & 31] = a;
  __syncthreads();
  if (r0 != 0 || col >= 2 * head_dim) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) a += red[i][threadIdx.x & 31];
  if (col < head_dim) {
    if (dq) dq[col] = a;
  } else if (dk) {
    dk[col - head_dim] = a;
  }
}

inline int qk_group(int head_dim) {
  int g = 2;
  while (g * 8 < head_dim) g *= 2;
  return g;
}
inline long long qk_blocks(long long M, int heads, int head_dim, bool grad, int sms) {
  const int s = 32 / qk_group(head_dim), chunks = (heads + s * QK_ROUNDS - 1) / (s * QK_ROUNDS);
  const long long blocks = (M * chunks + 7) / 8, cap = static_cast<long long>(sms) * (grad ? 4 : 16);
  return blocks < cap ? blocks : cap;
}

template <typename T, int G, bool GRAD>
inline int launch_qk_t(const QkParams& p, bool adjacent, unsigned blocks, cudaStream_t st) {
  return adjacent ? launch_chained(qk_norm_rope_kernel<T, G, true, GRAD>, dim3(blocks), 256, 0, st, 1, p)
                  : launch_chained(qk_norm_rope_kernel<T, G, false, GRAD>, dim3(blocks), 256, 0, st, 1, p);
}
template <typename T, bool GRAD>
inline int launch_qk_g(const QkParams& p, bool adjacent, unsigned blocks, cudaStream_t st) {
  switch (qk_group(p.head_dim)) {
    case 2: return launch_qk_t<T, 2, GRAD>(p, adjacent, blocks, st);
    case 4: return launch_qk_t<T, 4, GRAD>(p, adjacent, blocks, st);
    case 8: return launch_qk_t<T, 8, GRAD>(p, adjacent, blocks, st);
    case 16: return launch_qk_t<T, 16, GRAD>(p, adjacent, blocks, st);
    default: return launch_qk_t<T, 32, GRAD>(p, adjacent, blocks, st);
  }
}
template <bool GRAD>
inline int launch_qk(const QkParams& p, bool adjacent, bool fp16, long long blocks, cudaStream_t st) {
  return fp16 ? launch_qk_g<__half, GRAD>(p, adjacent, static_cast<unsigned>(blocks), st)
              : launch_qk_g<__nv_bfloat16, GRAD>(p, adjacent, static_cast<unsigned>(blocks), st);
}

}  // namespace strata
