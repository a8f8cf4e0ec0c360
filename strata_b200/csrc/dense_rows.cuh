// Row kernels of the dense layer: the forward pass for a few tokens, the gradient in front of the activation with its
// column sums, and the copy that gives rows of any width and stride whole 16-byte pieces.
#pragma once
#include "dense_tcgen05.cuh"

namespace strata {

// ---------------------------------------------------------------- y = r + act(x W^T + b) for 1 to 8 rows
// Bound by the weights' way from HBM (2 N K bytes; at one row an operation per byte), so no tensor cores: a 128-row
// tile would read the same bytes through N / 64 CTAs. A warp takes four output columns and all rows; its lanes have 16
// bytes of each of the four weight rows in flight at a time and share the x they multiply them with. kw of the block's
// eight warps split the contraction where N alone does not give every SM enough warps. Sums are fp32, even and odd k
// apart, then over the lanes and the kw warps in a fixed order.
constexpr int FEW_ROWS = 8;
constexpr int FEW_COLS = 4;

template <typename T, int VEC>
__device__ __forceinline__ void few_load(const T* p, uint64_t (&v)[VEC == 8 ? 4 : 1]) {
  if constexpr (VEC == 8) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    v[0] = pack2(Pair16<T>::lo(w.x), Pair16<T>::hi(w.x));
    v[1] = pack2(Pair16<T>::lo(w.y), Pair16<T>::hi(w.y));
    v[2] = pack2(Pair16<T>::lo(w.z), Pair16<T>::hi(w.z));
    v[3] = pack2(Pair16<T>::lo(w.w), Pair16<T>::hi(w.w));
  } else {
    v[0] = pack2(to_f32<T>(__ldg(p)), 0.f);
  }
}

template <typename T, int ROWS, int VEC>
__global__ void __launch_bounds__(256) dense_few_rows_kernel(const T* __restrict__ x, long long ldx,
                                                             const T* __restrict__ w, long long ldw, int kw,
                                                             const DenseParams p) {
  constexpr int NP = VEC == 8 ? 4 : 1, NV = FEW_COLS * ROWS;
  __shared__ float red[8][NV];
  chain_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / kw, part = warp - group * kw;
  const int col0 = (blockIdx.x * (8 / kw) + group) * FEW_COLS;
  uint64_t acc[FEW_COLS][ROWS];
#pragma unroll
  for (int c = 0; c < FEW_COLS; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) acc[c][r] = 0ull;
  const T* wr[FEW_COLS];
#pragma unroll
  for (int c = 0; c < FEW_COLS; ++c) wr[c] = w + min(col0 + c, p.N - 1) * ldw;
  const T* xr[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) xr[r] = x + min(r, p.M - 1) * ldx;
#pragma unroll(ROWS <= 2 ? 4 : 2)
  for (int k = (part * 32 + lane) * VEC; k < p.K; k += kw * 32 * VEC) {
    uint64_t wv[FEW_COLS][NP];
#pragma unroll
    for (int c = 0; c < FEW_COLS; ++c) few_load<T, VEC>(wr[c] + k, wv[c]);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint64_t xv[NP];
      few_load<T, VEC>(xr[r] + k, xv);
#pragma unroll
      for (int c = 0; c < FEW_COLS; ++c)
#pragma unroll
        for (int q = 0; q < NP; ++q) acc[c][r] = ffma2(wv[c][q], xv[q], acc[c][r]);
    }
  }
  float v[NV];
#pragma unroll
  for (int c = 0; c < FEW_COLS; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float lo, hi;
      unpack2(acc[c][r], lo, hi);
      v[c * ROWS + r] = lo + hi;
    }
  // over the lanes, halving what a lane keeps while there is something to halve: lane l ends up with value l / (32 / NV)
  int off = 16;
#pragma unroll
  for (int n = NV / 2; n >= 1; n >>= 1, off >>= 1) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const bool up = lane & off;
      const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
    }
  }
  for (; off >= 1; off >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
  constexpr int SHARE = 32 / NV;
  const int idx = lane / SHARE;
  if (lane % SHARE == 0) red[warp][idx] = v[0];
  __syncthreads();
  if (part != 0 || lane >= NV) return;
  float z = 0.f;
  for (int i = 0; i < kw; ++i) z += red[warp + i][lane];
  const int col = col0 + lane / ROWS, row = lane % ROWS;
  if (col >= p.N || row >= p.M) return;
  if (p.bias != nullptr) z += __ldg(p.bias + col);
  if (p.keep != nullptr) static_cast<T*>(p.keep)[row * p.ldk + col] = from_f32<T>(z);
  uint64_t y[1] = {pack2(z, 0.f)};
  dense_act<T>(p.act, y);
  float a, b;
  unpack2(y[0], a, b);
  if (p.aux != nullptr) a += to_f32<T>(static_cast<const T*>(p.aux)[row * p.ldaux + col]);
  static_cast<T*>(p.out)[row * p.ldo + col] = from_f32<T>(a);
}

// ---------------------------------------------------------------- dz = dy act'(z), and its column sums
// HBM-bound: reads dy and z, writes dz (act = none: reads dy, and writes it only where the products need aligned
// rows). A thread keeps its eight columns over all rows of the block, so the sums cost no extra read; the blocks' sums
// (fp32, of dz before it is rounded) are added up in a fixed order by dense_finish_kernel.
struct SlopeParams {
  const void* dy;  long long ldy;
  const void* z;   long long ldz;       // nullptr: act is none
  void* dz;        long long lddz;      // nullptr: sums only
  float* sums;                          // [gridDim.y, N] or nullptr
  int M, N, act, lanes, rows_per_block;   // lanes: threads along a row, a power of two
};

template <typename T, int VEC>
__device__ __forceinline__ void slope_load(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = Pair16<T>::lo(u[i]);
      v[2 * i + 1] = Pair16<T>::hi(u[i]);
    }
  } else {
    v[0] = to_f32<T>(__ldg(p));
  }
}

template <typename T, int VEC, int ACT>
__device__ __forceinline__ void slope_rows(const SlopeParams& p, int col, int r0, int step, int r1, float (&sum)[VEC]) {
  constexpr int U = 4;
  const T* dy = static_cast<const T*>(p.dy) + col;
  const T* z = static_cast<const T*>(p.z) + (ACT == ACT_NONE ? 0 : col);
  T* dz = static_cast<T*>(p.dz);
  for (int r = r0; r < r1; r += step * U) {
    float g[U][VEC], s[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = min(r + u * step, r1 - 1);
      slope_load<T, VEC>(dy + row * p.ldy, g[u]);
      if constexpr (ACT != ACT_NONE) slope_load<T, VEC>(z + row * p.ldz, s[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * step >= r1) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        // (not contracted into the sum: db has the same bits whether dz is stored or not)
        if constexpr (ACT != ACT_NONE) g[u][i] = __fmul_rn(g[u][i], dense_slope<ACT>(s[u][i]));
        sum[i] += g[u][i];
      }
      if (dz != nullptr) {
        T* to = dz + static_cast<long long>(r + u * step) * p.lddz + col;
        if constexpr (VEC == 8) {
          *reinterpret_cast<uint4*>(to) =
              make_uint4(Pair16<T>::pack(g[u][0], g[u][1]), Pair16<T>::pack(g[u][2], g[u][3]),
                         Pair16<T>::pack(g[u][4], g[u][5]), Pair16<T>::pack(g[u][6], g[u][7]));
        } else {
          *to = from_f32<T>(g[u][0]);
        }
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) dense_slope_kernel(const SlopeParams p) {
  __shared__ float red[256][VEC + (VEC > 1 ? 1 : 0)];
  chain_begin();
  const int lane = threadIdx.x & (p.lanes - 1), rr = threadIdx.x / p.lanes, step = 256 / p.lanes;
  const int col = (blockIdx.x * p.lanes + lane) * VEC;
  const long long b0 = static_cast<long long>(blockIdx.y) * p.rows_per_block;
  const int r1 = static_cast<int>(b0 + p.rows_per_block < p.M ? b0 + p.rows_per_block : p.M);
  float sum[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
  const bool live = col < p.N;
  if (live) {
    const int r0 = static_cast<int>(b0) + rr;
    switch (p.act) {
      case ACT_GELU: slope_rows<T, VEC, ACT_GELU>(p, col, r0, step, r1, sum); break;
      case ACT_GELU_TANH: slope_rows<T, VEC, ACT_GELU_TANH>(p, col, r0, step, r1, sum); break;
      case ACT_SILU: slope_rows<T, VEC, ACT_SILU>(p, col, r0, step, r1, sum); break;
      case ACT_RELU: slope_rows<T, VEC, ACT_RELU>(p, col, r0, step, r1, sum); break;
      default: slope_rows<T, VEC, ACT_NONE>(p, col, r0, step, r1, sum); break;
    }
  }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) red[threadIdx.x][i] = sum[i];
  __syncthreads();
  if (rr == 0 && live) {
    for (int k = 1; k < step; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] += red[k * p.lanes + lane][i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.sums[static_cast<long long>(blockIdx.y) * p.N + col + i] = sum[i];
  }
}

// ---------------------------------------------------------------- rows with whole 16-byte pieces
// Copies up to two matrices into rows whose stride is a multiple of 8 (what TMA reads). blockIdx.y: the matrix.
struct AlignRows {
  const uint16_t* src[2];
  uint16_t* dst[2];
  long long lds[2], ldd[2], rows[2];
  int cols[2];
};
__global__ void __launch_bounds__(256) dense_align_rows_kernel(const AlignRows a) {
  chain_begin();
  const int j = blockIdx.y;
  const uint16_t* __restrict__ src = a.src[j];
  uint16_t* __restrict__ dst = a.dst[j];
  const int cols = a.cols[j], nvec = static_cast<int>(a.ldd[j] >> 3);
  const long long n = a.rows[j] * nvec, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long t = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; t < n; t += step) {
    const long long row = t / nvec;
    const int c0 = static_cast<int>(t - row * nvec) * 8;
    const uint16_t* s = src + row * a.lds[j] + c0;
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? __ldg(s + i) : 0u;
    *reinterpret_cast<uint4*>(dst + row * a.ldd[j] + c0) =
        make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}

}  // namespace strata
