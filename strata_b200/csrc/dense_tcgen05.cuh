// The dense layer's products on the tensor cores: y = r + act(x W^T + b) and its gradients, bf16 or fp16 in and out,
// fp32 sums. The persistent, warp-specialised structure of gemm_tcgen05.cuh (TMA producer, MMA issuer, 16 epilogue
// warps, two accumulators in tensor memory, pairs of CTAs for large problems); what is new here:
//
//   layout    D[M, N] = A B with the operands as they lie in memory, never transposed by a pass of its own:
//               DENSE_NT   y = x W^T      A [M, K], B [N, K]   both rows run along the contraction ("K-major")
//               DENSE_NN   dx = dz W      A [M, K], B [K, N]   B's rows run across it ("MN-major")
//               DENSE_TN   dW = dz^T x    A [K, M], B [K, N]   both run across it
//             An MN-major tile is boxes of 64 x 64 (128 bytes of M or N, 64 contraction rows): the 128-byte-swizzled
//             layout the matrix descriptor names by its leading offset (from one box to the next) and its stride
//             (8 contraction rows).
//   epilogue  DENSE_Y: bias, activation, residual, one rounding; DENSE_Y_KEEP: z = x W^T + b besides;
//             DENSE_PART: fp32 partial sums of a split contraction (DensePlan), which dense_finish_kernel adds up
//             with the same epilogue.
//   widths    Rows of y and z that TMA cannot store (it writes whole 16-byte pieces) are copied from the staging boxes
//             by the warps.
#pragma once
#include "dense_common.cuh"
#include "gemm_tcgen05.cuh"

namespace strata {

enum DenseLayout : int { DENSE_NT = 0, DENSE_NN = 1, DENSE_TN = 2 };
enum DenseEpilogue : int { DENSE_Y = 0, DENSE_Y_KEEP = 1, DENSE_PART = 2 };

struct DenseParams {
  int M, N, K;                  // of the product: D [M, N], contraction K
  void* out;                    // D, 16-bit
  long long ldo;
  void* keep;                   // z or nullptr
  long long ldk;
  const void* aux;              // residual or nullptr
  long long ldaux;
  const float* bias;            // [N] or nullptr
  int act;
  int fp16;
  bool direct_out;              // out and keep are written by the warps, not by TMA
  bool direct_aux;              // the residual is read by the warps
  float* part;                  // DENSE_PART: slabs of TILE_M x BN
  const float* sums;            // column sums of dense_slope_kernel, [sum_rows, sum_cols], or nullptr; added up into
  int sum_rows, sum_cols;       //   db by epilogue warps that wait for their first tile
  float* db;
  DensePlan plan;
};

// db of eight columns: 256 threads, 32 rows of sums side by side, in a fixed order. `sync` is a barrier of those
// threads.
template <typename Sync>
__device__ __forceinline__ void dense_column_sums(const DenseParams& p, int group, int tid, float (*red)[9],
                                                  Sync sync) {
  const int col = group * 8 + (tid & 7), r0 = tid >> 3;
  float a = 0.f;
  if (col < p.sum_cols) {
#pragma unroll 8
    for (int r = r0; r < p.sum_rows; r += 32) a += p.sums[static_cast<long long>(r) * p.sum_cols + col];
  }
  red[r0][tid & 7] = a;
  sync();
  if (r0 == 0 && col < p.sum_cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) a += red[i][tid & 7];
    p.db[col] = a;
  }
}

// AHEAD: the residual of the next tile is loaded while this one is computed.
template <int BN, bool PAIR, int EPI, bool AHEAD>
struct DenseSmem {
  static constexpr int A_BYTES = GEMM_BM * GEMM_BK * 2;
  static constexpr int B_BYTES = (PAIR ? BN / 2 : BN) * GEMM_BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // staging boxes of a warp: 32 rows of 32 columns, or of all its columns of a tile
  static constexpr int BOX_COLS = AHEAD && BN == 256 ? 64 : 32;
  static constexpr int BOX_BYTES = 32 * BOX_COLS * 2;
  static constexpr int BOXES = EPI == DENSE_PART ? 0 : EPI == DENSE_Y_KEEP ? 2 : 1;
  static constexpr int STAGES = BN > 64 && BOXES * BOX_BYTES > 2048 ? 5 : 6;
  static constexpr int STAGING_OFF = STAGES * STAGE_BYTES;
  static constexpr int SUMS_BYTES = 32 * 9 * 4;                  // of dense_column_sums, in the boxes' place
  static constexpr int BAR_OFF = STAGING_OFF + (BOXES > 0 ? GEMM_EPI_WARPS * BOXES * BOX_BYTES : SUMS_BYTES);
  static constexpr int TOTAL = BAR_OFF + 512 + 1024;            // + alignment slack
  static_assert(TOTAL <= 232448, "shared memory of an SM");
};

// Descriptor of an operand tile: K-major as umma_smem_desc_sw128; MN-major with the 8192 bytes from one 64 x 64 box to
// the next as its leading offset.
__device__ __forceinline__ uint64_t dense_smem_desc(uint32_t addr, bool mn_major) {
  const uint64_t d = umma_smem_desc_sw128(addr);
  return mn_major ? (d & ~(0x3FFFull << 16)) | (static_cast<uint64_t>(8192 >> 4) << 16) : d;
}

// Pairs of values (two columns, the second one only if it exists) of rows with any alignment.
__device__ __forceinline__ void dense_store_pair(void* base, long long at, uint32_t w, bool two) {
  uint16_t* p = static_cast<uint16_t*>(base) + at;
  if (two && (reinterpret_cast<uintptr_t>(p) & 3u) == 0) {
    *reinterpret_cast<uint32_t*>(p) = w;
  } else {
    p[0] = static_cast<uint16_t>(w);
    if (two) p[1] = static_cast<uint16_t>(w >> 16);
  }
}
__device__ __forceinline__ uint32_t dense_load_pair(const void* base, long long at, bool two) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  if (two && (reinterpret_cast<uintptr_t>(p) & 3u) == 0) return *reinterpret_cast<const uint32_t*>(p);
  const uint32_t lo = *p;
  return two ? lo | (static_cast<uint32_t>(p[1]) << 16) : lo;
}
// A warp's copy of a 32 x 32 staging box (64-byte rows and swizzle) to rows that TMA does not store: two rows at a
// time, 16 lanes with neighbouring pairs each.
__device__ __forceinline__ void dense_copy_box(uint32_t box, void* base, long long ld, int m0, int n0, int M, int N) {
  const int lane = threadIdx.x & 31, j = lane & 15, col = n0 + 2 * j;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t r = 2 * i + (lane >> 4), piece = static_cast<uint32_t>(j >> 2) ^ ((r >> 1) & 3u);
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[i]) : "r"(box + r * 64u + (piece << 4) + (j & 3) * 4) : "memory");
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = m0 + 2 * i + (lane >> 4);
    if (row < M && col < N) dense_store_pair(base, static_cast<long long>(row) * ld + col, w[i], col + 1 < N);
  }
}

// Eight values of a row from p on, of which n exist (n <= 0: none), the others zero. ALIGNED: p is a multiple of 16
// bytes and n >= 8 or n <= 0. Otherwise the two aligned 16-byte pieces that hold them are read and shifted together: a
// piece is read only if it holds a value that exists, and memory is given out in larger units than 16 bytes.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load8(const void* p, int n) {
  uint4 u = make_uint4(0u, 0u, 0u, 0u);
  if (n <= 0) return u;
  if constexpr (ALIGNED) return __ldg(static_cast<const uint4*>(p));
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const int off = static_cast<int>(a & 15u) >> 1;
  const uint4* q = reinterpret_cast<const uint4*>(a & ~static_cast<uintptr_t>(15));
  const uint4 lo = __ldg(q);
  uint4 hi = u;
  if (off + (n < 8 ? n : 8) > 8) hi = __ldg(q + 1);
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (off & 4) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (off & 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const uint32_t bits = (off & 1) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
  if (n < 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i + 1 < n ? w[i] : (2 * i < n ? w[i] & 0xFFFFu : 0u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The way back, for rows that TMA does not load: 16-byte pieces, four lanes a row. alone: not a byte besides the box's
// own, in pairs (what is read is written by other warps meanwhile).
__device__ __forceinline__ void dense_load_box(uint32_t box, const void* base, long long ld, int m0, int n0, int M,
                                               int N, bool alone) {
  const int lane = threadIdx.x & 31;
  if (!alone) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + 8 * i + (lane >> 2), col = n0 + 8 * (lane & 3);
      v[i] = load8<false>(static_cast<const uint16_t*>(base) + static_cast<long long>(row < M ? row : m0) * ld + col,
                          N - col);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = 8 * i + (lane >> 2), piece = static_cast<uint32_t>(lane & 3) ^ ((r >> 1) & 3u);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + r * 64u + (piece << 4)), "r"(v[i].x),
                   "r"(v[i].y), "r"(v[i].z), "r"(v[i].w) : "memory");
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int j = lane & 15, row = m0 + 2 * i + (lane >> 4), col = n0 + 2 * j;
    const uint32_t r = 2 * i + (lane >> 4), piece = static_cast<uint32_t>(j >> 2) ^ ((r >> 1) & 3u);
    const uint32_t w =
        row < M && col < N ? dense_load_pair(base, static_cast<long long>(row) * ld + col, col + 1 < N) : 0u;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(box + r * 64u + (piece << 4) + (j & 3) * 4), "r"(w) : "memory");
  }
}

// Biases of this lane's column pairs in the 32 columns from n0 (zero behind column N).
__device__ __forceinline__ void dense_lane_bias(const DenseParams& p, int n0, int lane, uint64_t (&bias)[4]) {
  const int n = n0 + 2 * (lane & 3);
  if (p.bias != nullptr && n0 + 32 <= p.N && (reinterpret_cast<uintptr_t>(p.bias) & 7u) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = __ldg(reinterpret_cast<const unsigned long long*>(p.bias + n + 8 * i));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = n + 8 * i;
      bias[i] = p.bias == nullptr ? 0ull
                                  : pack2(k < p.N ? __ldg(p.bias + k) : 0.f, k + 1 < p.N ? __ldg(p.bias + k + 1) : 0.f);
    }
  }
}

// ACT: the activation, AUX: whether there is a residual; ACT_ANY: both, and how the rows are stored, are read from p.
template <int BN, bool PAIR, int LAY, int EPI, typename T, int ACT, bool AUX>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
dense_tcgen05_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmKeep,
                     const __grid_constant__ CUtensorMap tmAux, const DenseParams p) {
  constexpr bool AHEAD = AUX && EPI == DENSE_Y;
  using S = DenseSmem<BN, PAIR, EPI, AHEAD>;
  using P16 = Pair16<T>;
  constexpr bool A_MN = LAY == DENSE_TN, B_MN = LAY != DENSE_NT, PART = EPI == DENSE_PART, KEEP = EPI == DENSE_Y_KEEP;
  constexpr int TILE_M = PAIR ? 2 * GEMM_BM : GEMM_BM;
  constexpr bool ANY = ACT == ACT_ANY;
  const bool has_aux = ANY ? p.aux != nullptr : AUX, direct = ANY && p.direct_out;
  constexpr int BOX = 8192;                                // an MN-major box: 64 contraction rows of 128 bytes
  const uint32_t pair_rank = PAIR ? cluster_ctarank() : 0u;
  const int unit = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int n_units = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + S::BAR_OFF;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (S::STAGES + s); };
  auto accf_bar = [&](int b) { return bar_base + 8u * (2 * S::STAGES + b); };
  auto acce_bar = [&](int b) { return bar_base + 8u * (2 * S::STAGES + 2 + b); };
  auto aux_bar = [&](int w) { return bar_base + 8u * (2 * S::STAGES + 4 + w); };
  uint8_t* after = smem_gen + S::BAR_OFF + 8 * (2 * S::STAGES + 4 + GEMM_EPI_WARPS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(after);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(after + 8);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int tiles_m = (p.M + TILE_M - 1) / TILE_M;
  const int tiles_n = (p.N + BN - 1) / BN;
  const int num_tiles = tiles_m * tiles_n;
  const int num_kb = (p.K + GEMM_BK - 1) / GEMM_BK;
  // (the order of gemm_tcgen05_kernel: row block, then column tile)
  const bool ragged = p.N % BN != 0;
  auto tile_of = [&](int t, int& mt, int& jt) {
    mt = t / tiles_n;
    jt = t - mt * tiles_n;
    if (!PART && ragged) jt = (jt + static_cast<int>(static_cast<long long>(mt) * tiles_n / n_units)) % tiles_n;
  };
  auto tile_cols = [&](int j) { return min(BN, (p.N - j * BN + 31) / 32 * 32); };
  auto next = [&](DenseWalk& w, DenseSegment& g) -> bool {
    if constexpr (PART) {
      return w.next(p.plan, unit, g);
    } else {
      g = {w.t, 0, num_kb, 0};
      w.t += n_units;
      return g.tile < num_tiles;
    }
  };

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf_bar(b), 1);
      mbar_init(acce_bar(b), PAIR ? 2 * GEMM_EPI_WARPS : GEMM_EPI_WARPS);
    }
    for (int w = 0; w < GEMM_EPI_WARPS; ++w) mbar_init(aux_bar(w), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  chain_begin();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      DenseWalk walk(unit);
      DenseSegment g;
      while (ok && next(walk, g)) {
        int mt, jt;
        tile_of(g.tile, mt, jt);
        const int m0 = mt * TILE_M + static_cast<int>(pair_rank) * GEMM_BM;
        const int n0 = jt * BN + (PAIR ? static_cast<int>(pair_rank) * (tile_cols(jt) / 2) : 0);
        for (int kb = g.kb0; kb < g.kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, ST_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          const uint32_t a_dst = smem_base + stage * S::STAGE_BYTES;
          const uint32_t b_dst = a_dst + S::A_BYTES;
          // a pair's loads all complete on the first CTA's barrier, which announces the bytes of both
          const uint32_t fb = PAIR ? map_to_cta(full_bar(stage), 0) : full_bar(stage);
          if (!PAIR || pair_rank == 0) mbar_expect_tx(full_bar(stage), (PAIR ? 2 : 1) * S::STAGE_BYTES);
          auto load = [&](uint32_t dst, const CUtensorMap* tm, int x, int y) {
            if constexpr (PAIR) tma_load_2d_pair(dst, tm, x, y, fb);
            else tma_load_2d(dst, tm, x, y, fb);
          };
          if constexpr (A_MN) {
#pragma unroll
            for (int i = 0; i < S::A_BYTES / BOX; ++i) load(a_dst + i * BOX, &tmA, m0 + 64 * i, kb * GEMM_BK);
          } else {
            load(a_dst, &tmA, kb * GEMM_BK, m0);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int i = 0; i < S::B_BYTES / BOX; ++i) load(b_dst + i * BOX, &tmB, n0 + 64 * i, kb * GEMM_BK);
          } else {
            load(b_dst, &tmB, kb * GEMM_BK, n0);
          }
          if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        // Give loads already in flight time to land before the CTA retires.
#pragma unroll 1
        for (int i = 0; i < 2000; ++i) __nanosleep(100);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (pair_rank == 0 && elect_one()) {
      // (both operands have the launch's one type; the format fields are 1 for bf16 and 0 for fp16)
      uint32_t idesc0 = umma_idesc_bf16(TILE_M, 0, A_MN, B_MN);
      if (p.fp16) idesc0 &= ~((1u << 7) | (1u << 10));
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      DenseWalk walk(unit);
      DenseSegment g;
      for (; ok && next(walk, g); ++it) {
        int mt, jt;
        tile_of(g.tile, mt, jt);
        const uint32_t idesc = idesc0 | (static_cast<uint32_t>(tile_cols(jt) >> 3) << 17);
        const int buf = it & 1;
        if (!mbar_wait(acce_bar(buf), ((it >> 1) & 1u) ^ 1u, abort_flag, ST_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BN;
        for (int kb = g.kb0; kb < g.kb1; ++kb) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, ST_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_src = smem_base + stage * S::STAGE_BYTES;
          const uint64_t adesc = dense_smem_desc(a_src, A_MN);
          const uint64_t bdesc = dense_smem_desc(a_src + S::A_BYTES, B_MN);
#pragma unroll
          for (int k = 0; k < GEMM_BK / 16; ++k) {
            // 16 contraction values on: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
            const uint64_t a = adesc + (A_MN ? 128u : 2u) * k, b = bdesc + (B_MN ? 128u : 2u) * k;
            const uint32_t more = kb != g.kb0 || k != 0 ? 1u : 0u;
            if constexpr (PAIR) umma_ss_pair(d_tmem, a, b, idesc, more);
            else umma_ss(d_tmem, a, b, idesc, more);
          }
          if constexpr (PAIR) umma_commit_pair(empty_bar(stage)); else umma_commit(empty_bar(stage));
          if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok) {
          if constexpr (PAIR) umma_commit_pair(accf_bar(buf)); else umma_commit(accf_bar(buf));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue warps
    // Warp e has the 32 rows of its lane quarter and a quarter of the tile's columns, 32 at a time, as matrix fragments
    // (tmem_ld_16x256_x4): registers -> math -> staging box (swizzled) -> TMA store, clipped at the matrix's edge. The
    // residual is loaded into the box before; AHEAD, the box has all the warp's columns, and the next tile's residual
    // comes as soon as this tile's store has been read.
    const int e = warp - 2;
    const int quarter = warp & 3;
    const int cg = e >> 2;
    constexpr int WARP_COLS = BN < 128 ? 32 : BN / 4;
    constexpr int BC = S::BOX_COLS;
    const uint32_t acce_remote0 = PAIR ? map_to_cta(acce_bar(0), 0) : 0u;
    const uint32_t acce_remote1 = PAIR ? map_to_cta(acce_bar(1), 0) : 0u;
    [[maybe_unused]] const uint32_t box = smem_base + S::STAGING_OFF + e * S::BOXES * S::BOX_BYTES;
    [[maybe_unused]] const uint32_t zbox = box + S::BOX_BYTES;      // KEEP
    // this lane's row of the 8 x 8 pieces (rows 16 hf + {0, 8}, columns 32 c + 16 q + {0, 8}) of a box
    [[maybe_unused]] auto box_addr = [&](uint32_t b, int hf, int c, int q) -> uint32_t {
      const uint32_t r = ((lane >> 3) & 1) * 8 + (lane & 7), piece = 4 * c + 2 * q + (lane >> 4);
      return b + (16 * hf + r) * (BC * 2u) + ((BC == 64 ? piece ^ (r & 7) : piece ^ ((r >> 1) & 3)) << 4);
    };
    const bool load = !PART && ANY && has_aux && p.direct_aux, fetch = !PART && has_aux && !load;
    [[maybe_unused]] uint32_t aux_phase = 0;
    // first row and column of this warp's part of a tile; whether there is anything of it
    auto part_of = [&](int tile, int& m, int& n) -> bool {
      int mt, jt;
      tile_of(tile, mt, jt);
      m = mt * TILE_M + static_cast<int>(pair_rank) * GEMM_BM + quarter * 32;
      n = jt * BN + cg * WARP_COLS;
      return n < p.N && m < p.M && cg * WARP_COLS < BN;     // warp-uniform
    };
    [[maybe_unused]] auto fetch_aux = [&](int m, int n) {
      if (elect_one()) {
        tma_store_wait_read0();        // the box's last store has been read
        mbar_expect_tx(aux_bar(e), S::BOX_BYTES);
        tma_load_2d(box, &tmAux, n, m, aux_bar(e));
      }
    };
    if constexpr (LAY != DENSE_NT) {
      // the first eight warps, while the operands of the first tile are on their way
      if (p.sums != nullptr && e < 8) {
        float(*red)[9] = reinterpret_cast<float(*)[9]>(smem_gen + S::STAGING_OFF);
        auto sync = []() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        for (int group = blockIdx.x; group * 8 < p.sum_cols; group += gridDim.x) {
          dense_column_sums(p, group, static_cast<int>(threadIdx.x) - 64, red, sync);
          sync();
        }
      }
    }
    int it = 0;
    bool ok = true;
    DenseWalk walk(unit);
    DenseSegment g;
    if constexpr (AHEAD) {
      int m, n;
      if (unit < num_tiles && part_of(unit, m, n)) fetch_aux(m, n);
    }
    for (; ok && next(walk, g); ++it) {
      const int buf = it & 1;
      int m_warp, n_warp0;
      const bool live = part_of(g.tile, m_warp, n_warp0);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(buf * BN + cg * WARP_COLS);
      [[maybe_unused]] float* slab = nullptr;
      if constexpr (PART) {
        int mt, jt;
        tile_of(g.tile, mt, jt);
        slab = p.part + static_cast<long long>(g.slot) * (TILE_M * BN) +
               static_cast<long long>(m_warp - mt * TILE_M) * BN + (n_warp0 - jt * BN) + 2 * (lane & 3);
      }
      bool acc_ready = false;
#pragma unroll 1
      for (int c0 = 0; c0 < WARP_COLS; c0 += BC) {              // a box
        const bool box_live = live && n_warp0 + c0 < p.N;
        if (!AHEAD && fetch && box_live) fetch_aux(m_warp, n_warp0 + c0);
        if constexpr (ANY && !PART && BC == 32) {
          if (load && box_live) {
            if (elect_one()) tma_store_wait_read0();
            __syncwarp();
            dense_load_box(box, p.aux, p.ldaux, m_warp, n_warp0 + c0, p.M, p.N, p.aux == p.out);
            __syncwarp();
          }
        }
        if (!acc_ready) {
          if (!gemm_wait(accf_bar(buf), (it >> 1) & 1u, abort_flag, ST_TIMEOUT_EPILOGUE)) {
            ok = false;
            break;
          }
          tc_fence_after();
          acc_ready = true;
        }
        if (fetch && box_live) {
          if (!gemm_wait(aux_bar(e), aux_phase, abort_flag, ST_TIMEOUT_EPILOGUE)) {
            ok = false;
            break;
          }
          aux_phase ^= 1u;
        }
#pragma unroll 1
        for (int c = 0; c < BC / 32; ++c) {
          const int n0 = n_warp0 + c0 + 32 * c;
          const bool on = live && n0 < p.N;
          [[maybe_unused]] uint64_t bias[4];
          if constexpr (!PART) dense_lane_bias(p, n0, lane, bias);
          uint32_t acc[2][16];
          if (on) {
            tmem_ld_16x256_x4(taddr + c0 + 32 * c, acc[0]);
            tmem_ld_16x256_x4(taddr + c0 + 32 * c + (16u << 16), acc[1]);
            tmem_ld_wait();
          }
          if (c0 + 32 * c + 32 == WARP_COLS) {
            // the accumulator is in registers (or not needed): hand it back to the MMA warp
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) mbar_arrive_cluster(buf ? acce_remote1 : acce_remote0);
              else mbar_arrive(acce_bar(buf));
            }
          }
          if (!on) continue;
          // the fragment: pair i of half hf is row 16 hf + 8 (i % 2) + lane / 4, columns 8 (i / 2) + 2 (lane % 4)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            if constexpr (PART) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = 16 * hf + 8 * (i & 1) + (lane >> 2);
                if (m_warp + r < p.M)
                  *reinterpret_cast<uint2*>(slab + r * BN + c0 + 32 * c + 8 * (i >> 1)) =
                      make_uint2(acc[hf][2 * i], acc[hf][2 * i + 1]);
              }
            } else {
              uint64_t v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = fadd2(pack2u(acc[hf][2 * i], acc[hf][2 * i + 1]), bias[i >> 1]);
              auto put = [&](uint32_t b, bool wait) {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  float lo, hi;
                  unpack2(v[i], lo, hi);
                  w[i] = P16::pack(lo, hi);
                }
                if (wait && !direct) {      // as late as possible: the box's last store drains meanwhile
                  if (elect_one()) tma_store_wait_read0();
                  __syncwarp();
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) stmatrix_x4(box_addr(b, hf, c, q), &w[4 * q]);
              };
              if constexpr (KEEP) put(zbox, c == 0 && hf == 0 && !has_aux);
              if constexpr (LAY == DENSE_NT) {
                uint32_t aux[8];
                if (has_aux) {
#pragma unroll
                  for (int q = 0; q < 2; ++q) ldmatrix_x4(box_addr(box, hf, c, q), &aux[4 * q]);
                }
                if constexpr (ANY) dense_act<T>(p.act, v); else dense_act_all<T, ACT>(v);
                if (has_aux) {
#pragma unroll
                  for (int i = 0; i < 8; ++i) v[i] = fadd2(v[i], pack2(P16::lo(aux[i]), P16::hi(aux[i])));
                }
              }
              put(box, !KEEP && c == 0 && hf == 0 && !has_aux);
            }
          }
        }
        if (!PART && direct && box_live) {
          __syncwarp();
          if constexpr (KEEP) dense_copy_box(zbox, p.keep, p.ldk, m_warp, n_warp0 + c0, p.M, p.N);
          dense_copy_box(box, p.out, p.ldo, m_warp, n_warp0 + c0, p.M, p.N);
          __syncwarp();
        }
        if (!PART && !direct && box_live) {
          fence_proxy_async_smem();
          __syncwarp();
          if (elect_one()) {
            if constexpr (KEEP) tma_store_2d(&tmKeep, zbox, n_warp0 + c0, m_warp);
            tma_store_2d(&tmOut, box, n_warp0 + c0, m_warp);
            tma_store_commit();
          }
        }
      }
      if constexpr (AHEAD) {
        int m, n;
        if (ok && g.tile + n_units < num_tiles && part_of(g.tile + n_units, m, n)) fetch_aux(m, n);
      }
    }
    if (elect_one()) tma_store_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();   // no signal may reach a CTA that has already left
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ---------------------------------------------------------------- the second half of a split product
// Adds up a tile's slabs in a fixed order and applies the epilogue. A thread has four columns of a row; where a tile
// has many slabs, eight threads share them (64 x 64 of 64678 rows, 148 slabs: dW 30.7 us -> 15.8). Without slabs: the
// column sums alone (db where no product adds them up).
struct DenseFinish {
  DenseParams p;
  int tile_m, bn, tiles_n, blocks_per_tile, ways;
};

constexpr int FINISH_THREADS = 256;
constexpr int FINISH_SLOTS = 320;      // slabs of a tile: at most a unit's head and a helper's tail each

template <typename T>
__global__ void __launch_bounds__(FINISH_THREADS) dense_finish_kernel(const DenseFinish f) {
  chain_begin();
  const DenseParams& p = f.p;
  const DensePlan& s = p.plan;
  if (p.part == nullptr) {
    __shared__ float red[32][9];
    dense_column_sums(p, blockIdx.x, threadIdx.x, red, []() { __syncthreads(); });
    return;
  }
  __shared__ int slots[FINISH_SLOTS];
  __shared__ int n_slots;
  const int tile = blockIdx.x / f.blocks_per_tile;
  if (threadIdx.x == 0) {
    int n = 0;
    if (tile < s.whole) {
      slots[n++] = tile;
    } else {
      const int pieces = s.pieces();
      for (int c = 0; c < s.chunks; ++c) {
        const int v = c * s.rest + tile - s.whole;
        if (n < FINISH_SLOTS) slots[n++] = s.whole + v;
        if (s.tail > 0) {
          const long long x = static_cast<long long>(v) * s.tail;
          const int j1 = s.helper_of(x + s.tail - 1);
          for (int j = s.helper_of(x); j <= j1; ++j)
            if (n < FINISH_SLOTS) slots[n++] = s.whole + pieces + v + j;
        }
      }
    }
    n_slots = n;
  }
  __syncthreads();
  const int mt = tile / f.tiles_n, jt = tile - mt * f.tiles_n;
  const int per = FINISH_THREADS / f.ways, way = threadIdx.x / per;
  const int i = ((blockIdx.x - tile * f.blocks_per_tile) * per + threadIdx.x - way * per) * 4;
  const int r = i / f.bn, c = i - r * f.bn;
  const int row = mt * f.tile_m + r, col = jt * f.bn + c;
  const bool live = r < f.tile_m && row < p.M && col < p.N;
  if (f.ways == 1 && !live) return;
  const long long slab = static_cast<long long>(f.tile_m) * f.bn;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const int n = n_slots, share = (n + f.ways - 1) / f.ways, k1 = min(n, (way + 1) * share);
  if (live) {
#pragma unroll 4
    for (int k = way * share; k < k1; ++k) {
      const float4 b = *reinterpret_cast<const float4*>(p.part + slots[k] * slab + i);
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
  }
  if (f.ways > 1) {
    __shared__ float4 sums[FINISH_THREADS];
    sums[threadIdx.x] = a;
    __syncthreads();
    if (way > 0 || !live) return;
    for (int k = 1; k < f.ways; ++k) {
      const float4 b = sums[k * per + threadIdx.x];
      a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
  }
  float z[4] = {a.x, a.y, a.z, a.w};
  if (p.bias != nullptr) {
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] += col + k < p.N ? __ldg(p.bias + col + k) : 0.f;
  }
  uint64_t v[2] = {pack2(z[0], z[1]), pack2(z[2], z[3])};
  auto put = [&](void* base, long long ld) {
    const long long at = static_cast<long long>(row) * ld + col;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float lo, hi;
      unpack2(v[k], lo, hi);
      if (col + 2 * k < p.N) dense_store_pair(base, at + 2 * k, Pair16<T>::pack(lo, hi), col + 2 * k + 1 < p.N);
    }
  };
  if (p.keep != nullptr) put(p.keep, p.ldk);
  dense_act<T>(p.act, v);
  if (p.aux != nullptr) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (col + 2 * k < p.N) {
        const uint32_t w = dense_load_pair(p.aux, static_cast<long long>(row) * p.ldaux + col + 2 * k,
                                           col + 2 * k + 1 < p.N);
        v[k] = fadd2(v[k], pack2(Pair16<T>::lo(w), Pair16<T>::hi(w)));
      }
  }
  put(p.out, p.ldo);
}

}  // namespace strata
