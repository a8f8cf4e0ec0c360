// Row kernels of the dense layer: the forward pass for a few tokens, the gradient in front of the activation with its
// column sums, and the copy that gives rows of any width and stride whole 16-byte pieces.
#pragma once
#include "dense_tcgen05.cuh"

namespace strata {

// The epilogue for one output.
template <typename T>
__device__ __forceinline__ void dense_one(const DenseParams& p, int row, int col, float z) {
  if (row >= p.M || col >= p.N) return;
  if (p.bias != nullptr) z += __ldg(p.bias + col);
  if (p.keep != nullptr) static_cast<T*>(p.keep)[row * p.ldk + col] = from_f32<T>(z);
  uint64_t y[1] = {pack2(z, 0.f)};
  dense_act<T>(p.act, y);
  float a, b;
  unpack2(y[0], a, b);
  if (p.aux != nullptr) a += to_f32<T>(static_cast<const T*>(p.aux)[row * p.ldaux + col]);
  static_cast<T*>(p.out)[row * p.ldo + col] = from_f32<T>(a);
}

// ---------------------------------------------------------------- y = r + act(x W^T + b) for one to four rows
// Bound by the weights' way from HBM (2 N K bytes; at one row an operation per byte), so no tensor cores. A warp takes
// four output columns and all rows; its lanes have 16 bytes of each of the four weight rows in flight at a time, whole
// lines of a row, and share the x they multiply them with. kw of the block's eight warps split the contraction where N
// alone does not give every SM enough warps. Sums are fp32, even and odd k apart, then over the lanes and the kw warps
// in a fixed order.
constexpr int DOT_ROWS = 4;
constexpr int DOT_COLS = 4;

template <typename T>
__device__ __forceinline__ void dot_pairs(const uint4& u, uint64_t (&v)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack2(Pair16<T>::lo(w[i]), Pair16<T>::hi(w[i]));
}

template <typename T, int ROWS, bool ALIGNED>
__global__ void __launch_bounds__(256) dense_dot_rows_kernel(const T* __restrict__ x, long long ldx,
                                                             const T* __restrict__ w, long long ldw, int kw,
                                                             const DenseParams p) {
  constexpr int NV = DOT_COLS * ROWS;
  __shared__ float red[8][NV];
  chain_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / kw, part = warp - group * kw;
  const int col0 = (blockIdx.x * (8 / kw) + group) * DOT_COLS;
  uint64_t acc[DOT_COLS][ROWS];
#pragma unroll
  for (int c = 0; c < DOT_COLS; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) acc[c][r] = 0ull;
  // (columns and rows that do not exist repeat the last one)
  const T* wr[DOT_COLS];
#pragma unroll
  for (int c = 0; c < DOT_COLS; ++c) wr[c] = w + min(col0 + c, p.N - 1) * ldw;
  const T* xr[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) xr[r] = x + min(r, p.M - 1) * ldx;
#pragma unroll(ROWS <= 2 ? 4 : 2)
  for (int k = (part * 32 + lane) * 8; k < p.K; k += kw * 256) {
    uint4 raw[DOT_COLS];
#pragma unroll
    for (int c = 0; c < DOT_COLS; ++c) raw[c] = load8<ALIGNED>(wr[c] + k, p.K - k);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint64_t xv[4];
      dot_pairs<T>(load8<ALIGNED>(xr[r] + k, p.K - k), xv);
#pragma unroll
      for (int c = 0; c < DOT_COLS; ++c) {
        uint64_t wv[4];
        dot_pairs<T>(raw[c], wv);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[c][r] = ffma2(wv[q], xv[q], acc[c][r]);
      }
    }
  }
  float v[NV];
#pragma unroll
  for (int c = 0; c < DOT_COLS; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float lo, hi;
      unpack2(acc[c][r], lo, hi);
      v[c * ROWS + r] = lo + hi;
    }
  // over the lanes, halving what a lane keeps while there is something to halve: lane l ends up with value l / (32 /
  // NV)
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
  if (lane % SHARE == 0) red[warp][lane / SHARE] = v[0];
  __syncthreads();
  if (part != 0 || lane >= NV) return;
  float z = 0.f;
  for (int i = 0; i < kw; ++i) z += red[warp + i][lane];
  dense_one<T>(p, lane % ROWS, col0 + lane / ROWS, z);
}

// ---------------------------------------------------------------- y = r + act(x W^T + b) for a few rows
// Bound by the weights' way from HBM (2 N K bytes) and by latency: a 128-row tile on tcgen05 would read them through N
// / 64 CTAs and one pipeline each, or need a second kernel and a workspace to add up a split. Here a block has 16
// output columns and all rows; its eight warps, and where K is long the blocks of a cluster, split the contraction so
// that every warp has all it reads in flight at once. A lane reads 16 bytes of two weight rows and of a row of x
// straight into the fragments of mma.sync.m16n8k16: the product does not care which k is which as long as both
// operands agree, so lane t of a quad takes k = 8 t ... 8 t + 7 of 32 and hands them over as two steps of 16. Sums are
// fp32, over the warps and then over the cluster (through distributed shared memory) in a fixed order.
constexpr int FEW_ROWS = 32;
constexpr int FEW_COLS = 16;
constexpr int FEW_WARPS = 8;
constexpr int FEW_STEP = 32 * FEW_WARPS;      // contraction values that a block takes at a time

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if constexpr (Pair16<T>::UMMA_FORMAT == 1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// NT: blocks of eight rows. k_part: contraction values of a block of the cluster, a multiple of FEW_STEP.
template <typename T, int NT, bool ALIGNED>
__global__ void __launch_bounds__(32 * FEW_WARPS) dense_few_rows_kernel(const T* __restrict__ x, long long ldx,
                                                                        const T* __restrict__ w, long long ldw,
                                                                        int k_part, int parts, const DenseParams p) {
  constexpr int OUTS = 8 * NT * FEW_COLS;
  __shared__ float red[FEW_WARPS][8 * NT][FEW_COLS + 1];
  __shared__ float sum[OUTS];
  chain_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int col0 = blockIdx.x / parts * FEW_COLS;
  const int k0 = rank * k_part, k1 = min(p.K, k0 + k_part);
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  // (columns and rows that do not exist repeat the last one)
  const T* w0 = w + min(col0 + g, p.N - 1) * ldw + 8 * t;
  const T* w1 = w + min(col0 + g + 8, p.N - 1) * ldw + 8 * t;
  const T* xr[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) xr[i] = x + min(8 * i + g, p.M - 1) * ldx + 8 * t;
#pragma unroll(NT <= 2 ? 4 : 2)
  for (int k = k0 + warp * 32; k < k1; k += FEW_STEP) {
    const int n = p.K - k - 8 * t;
    const uint4 a = load8<ALIGNED>(w0 + k, n), b = load8<ALIGNED>(w1 + k, n);
    uint4 v[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) v[i] = load8<ALIGNED>(xr[i] + k, n);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      mma_16816<T>(acc[i], a.x, b.x, a.y, b.y, v[i].x, v[i].y);
      mma_16816<T>(acc[i], a.z, b.z, a.w, b.w, v[i].z, v[i].w);
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    red[warp][8 * i + 2 * t][g] = acc[i][0];
    red[warp][8 * i + 2 * t + 1][g] = acc[i][1];
    red[warp][8 * i + 2 * t][g + 8] = acc[i][2];
    red[warp][8 * i + 2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < OUTS; i += 32 * FEW_WARPS) {
    const int row = i / FEW_COLS, c = i % FEW_COLS;
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < FEW_WARPS; ++k) z += red[k][row][c];
    if (parts == 1) dense_one<T>(p, row, col0 + c, z);
    else sum[i] = z;
  }
  if (parts == 1) return;
  cluster_sync_all();
  // every block of the cluster finishes its share of the outputs
  for (int i = rank * 32 * FEW_WARPS + threadIdx.x; i < OUTS; i += parts * 32 * FEW_WARPS) {
    float z = 0.f;
    for (int k = 0; k < parts; ++k) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_u32(&sum[i]), k)) : "memory");
      z += v;
    }
    dense_one<T>(p, i / FEW_COLS, col0 + i % FEW_COLS, z);
  }
  cluster_sync_all();       // a block's sums are read until here
}

// ---------------------------------------------------------------- rows with whole 16-byte pieces
// Copies up to three matrices into rows whose stride is a multiple of 8 (what TMA reads), with zeros behind their
// columns. A block takes whole rows, `per` of them; a thread walks every 256th 16-byte piece, four in flight.
struct AlignRows {
  const uint16_t* src[3];
  uint16_t* dst[3];
  long long lds[3], ldd[3], rows[3];
  int cols[3], per[3];
  int n;
};
// Rows of a block: 512 to 2048 pieces, so that a small matrix has blocks for the whole chip (x of 10473 x 207 before a
// product: 19.6 us with 2048 pieces a block, 15.0 with 512; 12445 x 2873: 49 with 2048, 60 with 512).
inline int align_block_rows(long long rows, int cols, int sms) {
  const long long pieces = (cols + 7) / 8, share = rows * pieces / (8LL * sms);
  const long long n = (share < 512 ? 512 : share > 2048 ? 2048 : share) / pieces;
  return n > 0 ? static_cast<int>(n) : 1;
}
__device__ __forceinline__ void align_rows(const AlignRows& a, int j, int block, int blocks) {
  constexpr int U = 4;
  const int cols = a.cols[j], nvec = (cols + 7) / 8, per = a.per[j];
  const int dr = 256 / nvec, dc = 256 - dr * nvec, r_first = threadIdx.x / nvec, c_first = threadIdx.x - r_first * nvec;
  for (long long r0 = static_cast<long long>(block) * per; r0 < a.rows[j]; r0 += static_cast<long long>(blocks) * per) {
    const int rows = static_cast<int>(a.rows[j] - r0 < per ? a.rows[j] - r0 : per);
    const uint16_t* __restrict__ src = a.src[j] + r0 * a.lds[j];
    uint16_t* __restrict__ dst = a.dst[j] + r0 * a.ldd[j];
    int r = r_first, c = c_first;
    while (r < rows) {
      uint4 v[U];
      long long to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        to[u] = r < rows ? r * a.ldd[j] + c * 8 : -1;
        if (r < rows) v[u] = load8<false>(src + r * a.lds[j] + c * 8, cols - c * 8);
        r += dr;
        c += dc;
        if (c >= nvec) {
          c -= nvec;
          ++r;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (to[u] >= 0) *reinterpret_cast<uint4*>(dst + to[u]) = v[u];
    }
  }
}
__global__ void __launch_bounds__(256) dense_align_rows_kernel(const AlignRows a) {
  chain_begin();
  align_rows(a, blockIdx.y, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------- dz = dy act'(z), and its column sums
// HBM-bound: reads dy and z, writes dz (act = none: reads dy, and writes it only where the products need aligned
// rows). dz is rounded to the 16-bit type, which the tensor cores read: a second half of its digits would be a second
// product each for dx and dW (1024 x 512, K = 128: 0.24 % off 64 bits, 0.17 % with dz in 32). A thread keeps its eight
// columns over all rows of the block, so the sums cost no extra read; the blocks' sums (fp32, of dz before it is
// rounded) are added up in a fixed order by dense_finish_kernel.
struct SlopeParams {
  const void* dy;  long long ldy;
  const void* z;   long long ldz;       // nullptr: act is none
  void* dz;        long long lddz;      // nullptr: sums only
  float* sums;                          // [blocks / cols, N] or nullptr
  int M, N, act, lanes, rows_per_block;   // lanes: threads along a row, a power of two
  int cols, blocks, align_blocks;         // blocks along a row; of dz and the sums; of each matrix copied
};

template <typename T>
__device__ __forceinline__ void slope_unpack(const uint4& w, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = Pair16<T>::lo(u[i]);
    v[2 * i + 1] = Pair16<T>::hi(u[i]);
  }
}

template <typename T, bool ALIGNED, int ACT>
__device__ __forceinline__ void slope_rows(const SlopeParams& p, int col, int r0, int step, int r1, float (&sum)[8]) {
  constexpr int U = ALIGNED ? 4 : 2;      // rows in flight; of an unaligned one two pieces
  const T* dy = static_cast<const T*>(p.dy) + col;
  const T* z = static_cast<const T*>(p.z) + (ACT == ACT_NONE ? 0 : col);
  T* dz = static_cast<T*>(p.dz);
  for (int r = r0; r < r1; r += step * U) {
    uint4 g4[U], s4[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long row = min(r + u * step, r1 - 1);
      g4[u] = load8<ALIGNED>(dy + row * p.ldy, p.N - col);
      if constexpr (ACT != ACT_NONE) s4[u] = load8<ALIGNED>(z + row * p.ldz, p.N - col);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * step >= r1) break;
      float g[8], s[8];
      slope_unpack<T>(g4[u], g);
      if constexpr (ACT != ACT_NONE) slope_unpack<T>(s4[u], s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (not contracted into the sum: db has the same bits whether dz is stored or not)
        if constexpr (ACT != ACT_NONE) g[i] = __fmul_rn(g[i], dense_slope<ACT>(s[i]));
        sum[i] += g[i];
      }
      if (dz != nullptr)      // (rows of whole 16-byte pieces; zeros behind column N)
        *reinterpret_cast<uint4*>(dz + static_cast<long long>(r + u * step) * p.lddz + col) =
            make_uint4(Pair16<T>::pack(g[0], g[1]), Pair16<T>::pack(g[2], g[3]), Pair16<T>::pack(g[4], g[5]),
                       Pair16<T>::pack(g[6], g[7]));
    }
  }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) dense_slope_kernel(const SlopeParams p, const AlignRows a) {
  __shared__ float red[256][9];
  chain_begin();
  if (static_cast<int>(blockIdx.x) >= p.blocks) {
    const int b = blockIdx.x - p.blocks, j = b / p.align_blocks;
    align_rows(a, j, b - j * p.align_blocks, p.align_blocks);
    return;
  }
  const int block_y = blockIdx.x / p.cols, block_x = blockIdx.x - block_y * p.cols;
  const int lane = threadIdx.x & (p.lanes - 1), rr = threadIdx.x / p.lanes, step = 256 / p.lanes;
  const int col = (block_x * p.lanes + lane) * 8;
  const long long b0 = static_cast<long long>(block_y) * p.rows_per_block;
  const int r1 = static_cast<int>(b0 + p.rows_per_block < p.M ? b0 + p.rows_per_block : p.M);
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool live = col < p.N;
  if (live) {
    const int r0 = static_cast<int>(b0) + rr;
    switch (p.act) {
      case ACT_GELU: slope_rows<T, ALIGNED, ACT_GELU>(p, col, r0, step, r1, sum); break;
      case ACT_GELU_TANH: slope_rows<T, ALIGNED, ACT_GELU_TANH>(p, col, r0, step, r1, sum); break;
      case ACT_SILU: slope_rows<T, ALIGNED, ACT_SILU>(p, col, r0, step, r1, sum); break;
      case ACT_RELU: slope_rows<T, ALIGNED, ACT_RELU>(p, col, r0, step, r1, sum); break;
      default: slope_rows<T, ALIGNED, ACT_NONE>(p, col, r0, step, r1, sum); break;
    }
  }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[threadIdx.x][i] = sum[i];
  __syncthreads();
  if (rr == 0 && live) {
    for (int k = 1; k < step; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += red[k * p.lanes + lane][i];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < p.N) p.sums[static_cast<long long>(block_y) * p.N + col + i] = sum[i];
  }
}

}  // namespace strata
