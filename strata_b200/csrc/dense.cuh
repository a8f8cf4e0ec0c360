// Host side of the dense layer: which kernel, tile and split a product takes, its workspace, and the launches of a
// forward and a backward pass.
#pragma once
#include "dense_rows.cuh"

namespace strata {

// ---------------------------------------------------------------- tile and split of a product
struct DenseChoice {
  int bn;          // 64, 128: one CTA, 128 rows; 256: a pair of CTAs, 256 rows
  bool split;
  DensePlan plan;
  int tile_m() const { return bn == 256 ? 2 * GEMM_BM : GEMM_BM; }
  int64_t slab_bytes() const { return split ? static_cast<int64_t>(plan.slots()) * tile_m() * bn * 4 : 0; }
};

inline int dense_tiles(int M, int N, int bn) {
  const int tm = bn == 256 ? 2 * GEMM_BM : GEMM_BM;
  return ((M + tm - 1) / tm) * ((N + bn - 1) / bn);
}

// CTA pairs that are resident at once (not every SM has a partner), asked once per device.
inline int dense_pairs(int sms) {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms / 2;
  int fit = cached[dev].load(std::memory_order_relaxed);
  if (fit != 0) return fit;
  using S = DenseSmem<256, true, DENSE_Y, false>;
  auto kern = dense_tcgen05_kernel<256, true, DENSE_NT, DENSE_Y, __nv_bfloat16, ACT_ANY, false>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sms & ~1));
  cfg.blockDim = dim3(GEMM_THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&fit, kern, &cfg) != cudaSuccess || fit <= 0) {
    cudaGetLastError();
    return sms / 2;
  }
  if (fit > sms / 2) fit = sms / 2;
  cached[dev].store(fit, std::memory_order_relaxed);
  return fit;
}

// The cheapest form by a model of each one's time, in microseconds: a k-block of 64 on one unit, the part of a tile's
// epilogue that nothing hides, a launch, and a slab's way to memory and back. On 210 random products (40 to 100000
// rows, widths from 32 to 4000) the form it takes was within 1 % of the fastest on average, within 30 % in all. Some of
// the shapes it was checked on, tiles of 64 / 128 / 256 unsplit, then split (the one taken in brackets):
//   y   64 x 1024, K = 4096    12.0 / 13.5 / 23.3   [7.4] / 10.6 / 12.3
//   y   2500 x 650, K = 207    6.6 / [5.9] / 7.2    (no split: enough tiles, four k-blocks)
//   y   98304 x 512, K = 2048  255 / 187 / [153]    371 / 296 / 249
//   dW  512 x 128 of 65536 rows    161 / 176 / 182    [21.5] / 24.4 / 24.5
//   dW  1536 x 384 of 20000 rows   54 / 59 / 93       53 / [26.2] / 29.2
//   dW  2048 x 512 of 98304 rows   265 / 289 / 438    271 / 194 / [158]
//   dW  4096 x 4096 of 3000 rows   115 / 77 / [68]    156 / 77 / 97
inline DenseChoice dense_choice(int M, int N, int K, int sms) {
  const int num_kb = (K + GEMM_BK - 1) / GEMM_BK;
  DenseChoice best{};
  double best_us = 0.0;
  for (int bn = 64; bn <= 256; bn *= 2) {
    const int units = bn == 256 ? dense_pairs(sms) : sms, tiles = dense_tiles(M, N, bn);
    const double kb_us = bn == 256 ? 0.25 : bn == 128 ? 0.20 : 0.15;
    const double tile_us = bn == 256 ? 1.6 : bn == 128 ? 1.0 : 0.8;     // epilogue that nothing hides
    const int turns = (tiles + units - 1) / units;
    const double us = turns * (num_kb * kb_us > tile_us ? num_kb * kb_us : tile_us) + tile_us + 2.0;
    if (best.bn == 0 || us < best_us) {
      best = DenseChoice{bn, false, {}};
      best.plan.tiles = tiles;
      best.plan.units = units;
      best.plan.num_kb = num_kb;
      best_us = us;
    }
    const DensePlan s = dense_plan(tiles, units, num_kb, 4);
    if (s.rest == 0 || (s.chunks == 1 && s.tail == 0)) continue;
    const int tm = bn == 256 ? 2 * GEMM_BM : GEMM_BM;
    const double rows = static_cast<double>(M < tm ? M : tm) / tm;       // of a slab that exist
    const double slab_mb = s.slots() * rows * tm * bn * 4e-6;
    const int kbs = s.whole / units * num_kb + s.head;
    const double split_us = kbs * kb_us + tile_us + 2.0 + 1.7 + slab_mb * 2 / 6.0;
    if (split_us < 0.95 * best_us) {
      best = DenseChoice{bn, true, s};
      best_us = split_us;
    }
  }
  return best;
}

// ---------------------------------------------------------------- launches
struct DenseOperand {
  const void* p;
  long long ld;
  int readable = 0;      // columns that exist in memory, where they are more than the operand's (0: no more)
};

// Units that a product's kernel runs on, and its blocks.
inline int dense_grid(int tiles, int units, bool split) { return split || tiles >= units ? units : tiles; }
inline int dense_blocks(const DenseChoice& c) {
  return dense_grid(c.plan.tiles, c.plan.units, c.split) * (c.bn == 256 ? 2 : 1);
}

template <int BN, bool PAIR, int LAY, int EPI, typename T, int ACT = ACT_ANY, bool AUX = false>
inline int launch_dense_t(const DenseOperand& A, const DenseOperand& B, const DenseParams& p, int units,
                          cudaStream_t st) {
  const bool a_mn = LAY == DENSE_TN, b_mn = LAY != DENSE_NT;
  constexpr int TILE_M = PAIR ? 2 * GEMM_BM : GEMM_BM;
  CUtensorMap tmA, tmB, tmOut, tmKeep, tmAux;
  // (a box that a row ends in costs up to twice a whole one where the columns are the tile's rows or columns: there the
  // map has all that exist, and what they hold stays in outputs that nobody stores)
  auto mn_cols = [](const DenseOperand& o, int cols) { return o.readable > cols ? o.readable : cols; };
  auto map = [](CUtensorMap* tm, const DenseOperand& o, int rows, int cols, uint32_t bx, uint32_t by, TmapSwizzle sw) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(o.ld) * 2};
    const uint32_t box[2] = {bx, by};
    return make_tmap_bf16(tm, o.p, 2, dims, str, box, sw);      // (either 16-bit type: nothing is converted)
  };
  if (map(&tmA, A, a_mn ? p.K : p.M, a_mn ? mn_cols(A, p.M) : p.K, 64, a_mn ? 64 : GEMM_BM, TMAP_SWIZZLE_128B) != 0)
    return -20;
  if (map(&tmB, B, b_mn ? p.K : p.N, b_mn ? mn_cols(B, p.N) : p.K, 64, b_mn ? 64 : (PAIR ? BN / 2 : BN),
          TMAP_SWIZZLE_128B) != 0)
    return -21;
  tmOut = tmKeep = tmAux = tmA;
  using S = DenseSmem<BN, PAIR, EPI, AUX && EPI == DENSE_Y>;
  constexpr TmapSwizzle sw = S::BOX_COLS == 64 ? TMAP_SWIZZLE_128B : TMAP_SWIZZLE_64B;
  if (EPI != DENSE_PART && p.aux && !p.direct_aux &&
      map(&tmAux, {p.aux, p.ldaux}, p.M, p.N, S::BOX_COLS, 32, sw) != 0)
    return -23;
  if (EPI != DENSE_PART && !p.direct_out) {
    if (map(&tmOut, {p.out, p.ldo}, p.M, p.N, S::BOX_COLS, 32, sw) != 0) return -22;
    if (p.keep && map(&tmKeep, {p.keep, p.ldk}, p.M, p.N, S::BOX_COLS, 32, sw) != 0) return -25;
  }
  auto kern = dense_tcgen05_kernel<BN, PAIR, LAY, EPI, T, ACT, AUX>;
  static std::atomic<uint64_t> smem_set;
  if (const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), S::TOTAL, smem_set); e != cudaSuccess)
    return -static_cast<int>(e) - 1000;
  const int tiles = ((p.M + TILE_M - 1) / TILE_M) * ((p.N + BN - 1) / BN);
  // a split's units are its plan's: blocks that are not resident at once run one after the other, none waits
  // for another
  const int grid = dense_grid(tiles, units, EPI == DENSE_PART);
  return launch_chained(kern, dim3(static_cast<unsigned>(PAIR ? 2 * grid : grid)), GEMM_THREADS, S::TOTAL, st,
                        PAIR ? 2 : 1, tmA, tmB, tmOut, tmKeep, tmAux, p);
}

// Forward pass on pairs of CTAs: a kernel for each activation, with and without a residual. One kernel that reads both
// from its parameters keeps the registers and the code of all of them in its loop; 262144 x 2048, K = 512, microseconds
// that way / this: no activation 431 / 415, silu 539 / 435, gelu (a longer formula then) 673 / 481, with a residual
// 658 / 590. The residual a tile ahead, in boxes of 64 columns: 590 -> 537; such boxes without a residual: silu 435 ->
// 497.
template <int EPI, typename T, bool AUX>
inline int launch_dense_pair(const DenseOperand& A, const DenseOperand& B, const DenseParams& p, int units,
                             cudaStream_t st) {
  switch (p.act) {
    case ACT_GELU: return launch_dense_t<256, true, DENSE_NT, EPI, T, ACT_GELU, AUX>(A, B, p, units, st);
    case ACT_GELU_TANH: return launch_dense_t<256, true, DENSE_NT, EPI, T, ACT_GELU_TANH, AUX>(A, B, p, units, st);
    case ACT_SILU: return launch_dense_t<256, true, DENSE_NT, EPI, T, ACT_SILU, AUX>(A, B, p, units, st);
    case ACT_RELU: return launch_dense_t<256, true, DENSE_NT, EPI, T, ACT_RELU, AUX>(A, B, p, units, st);
    default: return launch_dense_t<256, true, DENSE_NT, EPI, T, ACT_NONE, AUX>(A, B, p, units, st);
  }
}

template <int LAY, int EPI, typename T>
inline int launch_dense_bn(int bn, const DenseOperand& A, const DenseOperand& B, const DenseParams& p, int units,
                           cudaStream_t st) {
  if constexpr (LAY == DENSE_NT && EPI != DENSE_PART) {
    if (bn == 256 && !p.direct_out && !p.direct_aux)
      return p.aux ? launch_dense_pair<EPI, T, true>(A, B, p, units, st)
                   : launch_dense_pair<EPI, T, false>(A, B, p, units, st);
  }
  if (bn == 256) return launch_dense_t<256, true, LAY, EPI, T>(A, B, p, units, st);
  if (bn == 128) return launch_dense_t<128, false, LAY, EPI, T>(A, B, p, units, st);
  return launch_dense_t<64, false, LAY, EPI, T>(A, B, p, units, st);
}

inline int launch_dense_finish(const DenseFinish& f, cudaStream_t st) {
  const int blocks = f.p.part ? f.p.plan.tiles * f.blocks_per_tile : (f.p.sum_cols + 7) / 8;
  if (f.p.fp16)
    return launch_chained(dense_finish_kernel<__half>, dim3(blocks), FINISH_THREADS, 0, st, 1, f);
  return launch_chained(dense_finish_kernel<__nv_bfloat16>, dim3(blocks), FINISH_THREADS, 0, st, 1, f);
}

// One product of a choice, with the second kernel where it is split.
template <int LAY>
inline int launch_dense(const DenseOperand& A, const DenseOperand& B, DenseParams p, const DenseChoice& c, void* slabs,
                        cudaStream_t st) {
  if (!c.split) {
    if (LAY == DENSE_NT && p.keep != nullptr)
      return p.fp16 ? launch_dense_bn<DENSE_NT, DENSE_Y_KEEP, __half>(c.bn, A, B, p, c.plan.units, st)
                    : launch_dense_bn<DENSE_NT, DENSE_Y_KEEP, __nv_bfloat16>(c.bn, A, B, p, c.plan.units, st);
    return p.fp16 ? launch_dense_bn<LAY, DENSE_Y, __half>(c.bn, A, B, p, c.plan.units, st)
                  : launch_dense_bn<LAY, DENSE_Y, __nv_bfloat16>(c.bn, A, B, p, c.plan.units, st);
  }
  p.part = static_cast<float*>(slabs);
  p.plan = c.plan;
  // (the slabs are fp32 and the type is a bit of the instruction descriptor: one kernel for both)
  if (const int r = launch_dense_bn<LAY, DENSE_PART, __nv_bfloat16>(c.bn, A, B, p, c.plan.units, st); r != 0) return r;
  DenseFinish f{};
  f.p = p;
  f.tile_m = c.tile_m();
  f.bn = c.bn;
  f.tiles_n = (p.N + c.bn - 1) / c.bn;
  const int rows = p.M < f.tile_m ? p.M : f.tile_m;        // of a slab that exist
  f.ways = c.plan.slots() >= 16 * c.plan.tiles ? 8 : 1;
  f.blocks_per_tile = (rows * c.bn * f.ways + 4 * FINISH_THREADS - 1) / (4 * FINISH_THREADS);
  return launch_dense_finish(f, st);
}

// Few rows: dot products up to DOT_ROWS, else mma.sync.
template <typename T, bool ALIGNED>
inline int launch_few_rows_t(const DenseOperand& x, const DenseOperand& w, const DenseParams& p, int sms,
                             cudaStream_t st) {
  const T* xp = static_cast<const T*>(x.p);
  const T* wp = static_cast<const T*>(w.p);
  if (p.M <= DOT_ROWS) {
    // warps: four columns each, split along the contraction until every SM has eight
    const int groups = (p.N + DOT_COLS - 1) / DOT_COLS;
    int kw = 1;
    while (kw < 8 && groups * kw < 8 * sms && p.K >= 512 * kw) kw *= 2;
    const dim3 grid(static_cast<unsigned>((groups + 8 / kw - 1) / (8 / kw)));
    auto go = [&](auto kern) { return launch_chained(kern, grid, 256, 0, st, 1, xp, x.ld, wp, w.ld, kw, p); };
    if (p.M == 1) return go(dense_dot_rows_kernel<T, 1, ALIGNED>);
    if (p.M == 2) return go(dense_dot_rows_kernel<T, 2, ALIGNED>);
    return go(dense_dot_rows_kernel<T, 4, ALIGNED>);
  }
  // a cluster along the contraction where a warp would make more than two steps of it
  const int blocks = (p.N + FEW_COLS - 1) / FEW_COLS, steps = (p.K + FEW_STEP - 1) / FEW_STEP;
  int parts = 1;
  while (parts < 8 && steps > 2 * parts && 2 * parts * blocks <= 8 * sms) parts *= 2;
  const int k_part = (steps + parts - 1) / parts * FEW_STEP;
  auto go = [&](auto kern) {
    return launch_chained(kern, dim3(static_cast<unsigned>(blocks * parts)), 32 * FEW_WARPS, 0, st, parts, xp, x.ld, wp,
                          w.ld, k_part, parts, p);
  };
  if (p.M <= 8) return go(dense_few_rows_kernel<T, 1, ALIGNED>);
  if (p.M <= 16) return go(dense_few_rows_kernel<T, 2, ALIGNED>);
  return go(dense_few_rows_kernel<T, 4, ALIGNED>);
}
inline int launch_few_rows(const DenseOperand& x, const DenseOperand& w, const DenseParams& p, bool aligned, int sms,
                           cudaStream_t st) {
  if (p.fp16)
    return aligned ? launch_few_rows_t<__half, true>(x, w, p, sms, st)
                   : launch_few_rows_t<__half, false>(x, w, p, sms, st);
  return aligned ? launch_few_rows_t<__nv_bfloat16, true>(x, w, p, sms, st)
                 : launch_few_rows_t<__nv_bfloat16, false>(x, w, p, sms, st);
}

// Whether the forms for a few rows take a product: one launch and no workspace. From nine rows on every block of 16
// columns reads more of x than of W, and the tiles of a split product overtake them at large weights. Microseconds of
// these / of a split, weights out of HBM (half, gelu, residual): 9 x 1024, K = 1024 3.8 / 5.8; 16 x 2048, K = 2048 6.0
// / 10.6; 24 x 1024, K = 4096 8.0 / 8.5; 24 x 4096, K = 1024 7.7 / 8.4; 32 x 512, K = 2048 5.2 / 7.8; 32 x 4096, K =
// 4096 21.9 / 13.6; 48 x 1024, K = 4096 16.2 / 8.7; 8 x 4096, K = 4096 13.3 / 14.0. Dot products / mma.sync: 1 x 4096,
// K = 1024 4.3 / 5.0; 1 x 1024, K = 4096 4.1 / 7.8; 4 x 4096, K = 1024 4.9 / 5.0; 8 x 4096, K = 1024 12.7 / 5.0.
inline bool dense_few(int M, int N, int K) {
  const long long weights = static_cast<long long>(N) * K;
  return M <= 8 || (M <= FEW_ROWS && (M <= 16 ? 2 : 4) * weights <= (1ll << 25));
}

// Row stride of what the layer lays out for itself: whole 128-byte lines (or a part of one that holds the row). TMA's
// boxes are 128 bytes wide, and each of their rows that straddles two lines is two requests: dW 1080 x 632 of 18159
// rows 48 us with both operands' rows on any 16 bytes, 42 with dz's on lines, 38 with both; dx 18159 x 632 of 1080
// columns 31, 26, 25; y 20000 x 2040 of 520 columns 55, 48 (x on lines), 41.
inline int dense_pitch(int n) { return n <= 16 ? 16 : n <= 32 ? 32 : (n + 63) / 64 * 64; }
inline bool dense_aligned(const void* p, long long ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0;
}
// Rows that TMA may store: it writes whole 16-byte pieces, with zeros behind the last column. padded: those are the
// caller's to write.
inline bool dense_whole(const void* p, long long ld, int cols, bool padded) {
  return dense_aligned(p, ld) && (cols % 8 == 0 || padded);
}

// Pieces of a workspace, 256-byte aligned.
struct DenseArena {
  uint8_t* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

// Adds a copy of o to a and makes o the copy.
inline void align_add(AlignRows& a, DenseOperand& o, void* to, long long rows, int cols, int sms) {
  const int ld = dense_pitch(cols);
  const int n = a.n++;
  a.src[n] = static_cast<const uint16_t*>(o.p); a.lds[n] = o.ld;
  a.dst[n] = static_cast<uint16_t*>(to); a.ldd[n] = ld;
  a.rows[n] = rows; a.cols[n] = cols; a.per[n] = align_block_rows(rows, cols, sms);
  o = {to, ld, ld};
}
inline int align_blocks(const AlignRows& a, int sms) {       // of one matrix
  long long most = 0;
  for (int j = 0; j < a.n; ++j) {
    const long long blocks = (a.rows[j] + a.per[j] - 1) / a.per[j];
    most = blocks > most ? blocks : most;
  }
  return static_cast<int>(most < 8LL * sms ? most : 8LL * sms);
}

// ---------------------------------------------------------------- forward
// A residual that TMA cannot read is read by the epilogue's warps, or copied where a kernel for copies runs anyway and
// units have several tiles (which hide a TMA load better). Read / copied, microseconds: 10473 x 650, K = 207 24.0 /
// 22.7 (half); 30000 x 1001, K = 207 78 / 73; 40000 x 250, K = 77 25 / 28; 2500 x 650, K = 207 11.4 / 14.1; x aligned:
// 10473 x 650, K = 208 18 / 22; 24000 x 105, K = 40 15 / 30; 61552 x 97, K = 552 29 / 41; 16899 x 913, K = 3448 105 /
// 116; 20000 x 2047, K = 512 92 / 91; 120828 x 1428, K = 40 308 / 294.
inline bool dense_copies_residual(const DenseChoice& c, bool x_ok, bool w_ok, bool r_ok) {
  return !r_ok && !(x_ok && w_ok) && c.plan.tiles > c.plan.units;
}
// Workspace: aligned copies of the operands that are not aligned themselves, then the slabs of a split.
inline int64_t dense_forward_bytes(int M, int N, int K, bool x_ok, bool w_ok, bool r_ok, int sms) {
  if (dense_few(M, N, K)) return 0;
  DenseArena ws{nullptr, 0};
  const DenseChoice c = dense_choice(M, N, K, sms);
  if (!x_ok) ws.take(2LL * dense_pitch(K) * M);
  if (!w_ok) ws.take(2LL * dense_pitch(K) * N);
  if (dense_copies_residual(c, x_ok, w_ok, r_ok)) ws.take(2LL * dense_pitch(N) * M);
  ws.take(c.slab_bytes());
  return ws.used;
}

inline int launch_dense_forward(DenseOperand x, DenseOperand w, DenseParams p, void* workspace, int sms,
                                cudaStream_t st) {
  const bool x_ok = dense_aligned(x.p, x.ld), w_ok = dense_aligned(w.p, w.ld);
  if (dense_few(p.M, p.N, p.K)) return launch_few_rows(x, w, p, x_ok && w_ok && p.K % 8 == 0, sms, st);
  DenseArena ws{static_cast<uint8_t*>(workspace), 0};
  AlignRows a{};
  if (!x_ok) align_add(a, x, ws.take(2LL * dense_pitch(p.K) * p.M), p.M, p.K, sms);
  if (!w_ok) align_add(a, w, ws.take(2LL * dense_pitch(p.K) * p.N), p.N, p.K, sms);
  const DenseChoice c = dense_choice(p.M, p.N, p.K, sms);
  p.direct_aux = p.aux && !dense_aligned(p.aux, p.ldaux);
  if (dense_copies_residual(c, x_ok, w_ok, !p.direct_aux)) {
    DenseOperand r{p.aux, p.ldaux};
    align_add(a, r, ws.take(2LL * dense_pitch(p.N) * p.M), p.M, p.N, sms);
    p.aux = r.p;
    p.ldaux = r.ld;
    p.direct_aux = false;
  }
  if (a.n > 0) {
    const dim3 grid(static_cast<unsigned>(align_blocks(a, sms)), static_cast<unsigned>(a.n));
    if (const int r = launch_chained(dense_align_rows_kernel, grid, 256, 0, st, 1, a); r != 0) return r;
  }
  return launch_dense<DENSE_NT>(x, w, p, c, ws.take(c.slab_bytes()), st);
}

// ---------------------------------------------------------------- backward
struct DenseGradParams {
  int M, N, K, act, fp16;
  bool padded;                     // dx may be written up to whole 16-byte pieces of its rows
  DenseOperand dy, x, w, z;        // z.p nullptr: act is none
  void* dx; long long lddx;        // any of the three outputs may be absent
  void* dw; long long lddw;
  float* db;
};

struct DenseGradSums { int lanes, cols, rows_per_block, blocks; };     // geometry of dense_slope_kernel

inline DenseGradSums dense_grad_sums(int M, int N, int sms) {
  DenseGradSums g{};
  const int units = (N + 7) / 8;
  g.lanes = 1;
  while (g.lanes < 32 && g.lanes < units) g.lanes *= 2;
  g.cols = (units + g.lanes - 1) / g.lanes;
  const int step = 256 / g.lanes;
  // eight blocks of 256 threads on every SM, but no fewer than four rows a thread
  long long blocks = (8LL * sms + g.cols - 1) / g.cols;
  const long long most = (M + 4LL * step - 1) / (4LL * step);
  if (blocks > most) blocks = most;
  g.rows_per_block = static_cast<int>((M + blocks - 1) / blocks);
  g.blocks = static_cast<int>((M - 1LL + g.rows_per_block) / g.rows_per_block);     // (the sum may leave 32 bits)
  return g;
}

// dz goes through memory when there is an activation, or when dy is not aligned; then its rows are dense_pitch(N)
// apart.
struct DenseGradPlan {
  bool copy_x, copy_w, make_dz, aligned;
  DenseChoice cx, cw;
  DenseGradSums sums;
  int64_t bytes;
  void *dz, *xs, *ws, *slabs;
  float* col_sums;
};

inline DenseGradPlan dense_grad_plan(int M, int N, int K, bool act, bool dy_ok, bool z_ok, bool x_ok, bool w_ok,
                                     bool dx, bool dw, bool db, void* workspace, int sms) {
  DenseGradPlan g{};
  g.make_dz = (dx || dw) && (act || !dy_ok);
  g.copy_x = dw && !x_ok;
  g.copy_w = dx && !w_ok;
  g.aligned = dy_ok && (!act || z_ok) && N % 8 == 0;
  g.sums = dense_grad_sums(M, N, sms);
  if (dx) g.cx = dense_choice(M, K, N, sms);
  if (dw) g.cw = dense_choice(N, K, M, sms);
  DenseArena ws{static_cast<uint8_t*>(workspace), 0};
  if (g.make_dz) g.dz = ws.take(2LL * dense_pitch(N) * M);
  if (g.copy_x) g.xs = ws.take(2LL * dense_pitch(K) * M);
  if (g.copy_w) g.ws = ws.take(2LL * dense_pitch(K) * N);
  if (db && g.sums.blocks > 1) g.col_sums = static_cast<float*>(ws.take(4LL * g.sums.blocks * N));
  const int64_t sx = g.cx.slab_bytes(), sw = g.cw.slab_bytes();
  g.slabs = ws.take(sx > sw ? sx : sw);        // one after the other on the stream
  g.bytes = ws.used;
  return g;
}

inline int launch_dense_backward(const DenseGradParams& q, const DenseGradPlan& g, int sms, cudaStream_t st) {
  DenseOperand x = q.x, w = q.w, dz = q.dy;
  int r;
  AlignRows a{};
  if (g.copy_x) align_add(a, x, g.xs, q.M, q.K, sms);
  if (g.copy_w) align_add(a, w, g.ws, q.N, q.K, sms);
  if (g.make_dz || q.db || a.n > 0) {
    SlopeParams s{};
    s.dy = q.dy.p; s.ldy = q.dy.ld;
    s.z = q.z.p; s.ldz = q.z.ld;
    s.dz = g.make_dz ? g.dz : nullptr; s.lddz = dense_pitch(q.N);
    s.sums = g.sums.blocks == 1 ? q.db : g.col_sums;
    s.M = q.M; s.N = q.N; s.act = q.act; s.lanes = g.sums.lanes; s.rows_per_block = g.sums.rows_per_block;
    s.cols = g.sums.cols;
    s.blocks = g.make_dz || q.db ? g.sums.cols * g.sums.blocks : 0;
    s.align_blocks = align_blocks(a, sms);
    const dim3 grid(static_cast<unsigned>(s.blocks + s.align_blocks * a.n));
    auto go = [&](auto kern) { return launch_chained(kern, grid, 256, 0, st, 1, s, a); };
    if (q.fp16) r = g.aligned ? go(dense_slope_kernel<__half, true>) : go(dense_slope_kernel<__half, false>);
    else r = g.aligned ? go(dense_slope_kernel<__nv_bfloat16, true>) : go(dense_slope_kernel<__nv_bfloat16, false>);
    if (r != 0) return r;
    if (g.make_dz) dz = {g.dz, dense_pitch(q.N), dense_pitch(q.N)};
  }
  // db is added up by the first product's kernel, unless the product has too few blocks for it (2 x 16 x 472: 31 us in
  // the one block of dx, 4 in a kernel of its own). The sums of a single block of rows are db.
  auto sums = [&](DenseParams& p) {
    p.sums = g.col_sums; p.sum_rows = g.sums.blocks; p.sum_cols = q.N; p.db = q.db;
  };
  const int groups = q.db && g.sums.blocks > 1 ? (q.N + 7) / 8 : 0;
  const bool in_dx = q.dx && groups > 0 && groups <= 4 * dense_blocks(g.cx);
  const bool in_dw = !q.dx && q.dw && groups > 0 && groups <= 4 * dense_blocks(g.cw);
  if (groups > 0 && !in_dx && !in_dw) {
    DenseFinish f{};
    sums(f.p);
    f.p.fp16 = q.fp16;
    if ((r = launch_dense_finish(f, st)) != 0) return r;
  }
  if (q.dx) {
    DenseParams p{};
    p.M = q.M; p.N = q.K; p.K = q.N;
    p.out = q.dx; p.ldo = q.lddx; p.fp16 = q.fp16;
    p.direct_out = !dense_whole(q.dx, q.lddx, q.K, q.padded);
    if (in_dx) sums(p);
    if ((r = launch_dense<DENSE_NN>(dz, w, p, g.cx, g.slabs, st)) != 0) return r;
  }
  if (q.dw) {
    DenseParams p{};
    p.M = q.N; p.N = q.K; p.K = q.M;
    p.out = q.dw; p.ldo = q.lddw; p.fp16 = q.fp16;
    p.direct_out = !dense_whole(q.dw, q.lddw, q.K, false);
    if (in_dw) sums(p);
    return launch_dense<DENSE_TN>(dz, x, p, g.cw, g.slabs, st);
  }
  return 0;
}

}  // namespace strata
