// Persistent warp-specialised tcgen05 GEMM over groups of rows (one group per
// expert), bf16 operands and fp32 accumulation in TMEM.  Group g holds the
// rows [offsets[g], offsets[g+1]) of the row operands and has its own weight
// matrix W_g [N, K]:
//
//   kForward   Y[r, n]    = sum_k X[r, k] W_g[n, k]       (X K-major, W K-major)
//   kDataGrad  dX[r, k]   = sum_n dY[r, n] W_g[n, k]      (dY K-major, W MN-major)
//   kWeightGrad dW_g[n,k] = sum_{r in g} dY[r, n] X[r, k] (both MN-major)
//
// The offsets are read on the device, so nothing is known on the host but the
// total number of rows.  Every CTA copies them into shared memory, checks them
// against the rows that exist and scans the groups' tile counts once; a tile
// index is then found by binary search.
//
// A tile of a group's last rows also loads rows of the next group; they only
// reach accumulator rows that are never stored.  Stores: 32-row slabs that
// belong to the group whole leave by TMA, the group's last slab row by row.
// In the weight gradient the rows are the summed dimension: the last 64-row
// step of a group whose size is not a multiple of 64 is fetched apart (onto a
// barrier of this CTA), and the producer warp writes zeros over the foreign
// rows of both operands before the MMA may read the step -- a foreign row may
// hold NaN, so zeroing one operand would not do.  In the MN-major layout a row
// is a 128-byte line of each 64-column box, so the zeros need no swizzle.
//
// Roles and barriers are those of gemm.cuh (CG = 1: 128 x BN tiles) and
// gemm2.cuh (CG = 2: 256 x 256 tiles on SM pairs): warp 0 TMA producer, warp 1
// MMA issuer, warps 2..5 epilogue; all waits are bounded.
#pragma once
#include "gemm.cuh"
#include "gemm2.cuh"
#include "gemm_epi.cuh"

namespace tdb {
namespace grouped {

using gemm::BK;
constexpr int kThreads = 192;
constexpr int kMaxGroups = 1024;

enum Op : int { kForward = 0, kDataGrad = 1, kWeightGrad = 2 };

template <int CG, int BN>
struct Config {
  static constexpr int kTileM = 128 * CG;      // output rows per tile (128 per CTA)
  static constexpr int kBRows = BN / CG;       // output columns whose operand rows this CTA stages
  static constexpr int kABytes = 128 * BK * 2;
  static constexpr int kBBytes = kBRows * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 5;
  static constexpr int kTmemCols = 2 * BN;     // two accumulators
  static constexpr int kEpiBuf = 4096;         // one staged block of an epilogue warp
  static constexpr int kEpiBytes = 4 * 2 * kEpiBuf;
  static constexpr int kBarBytes = 256;
  static_assert(kTmemCols == 256 || kTmemCols == 512, "TMEM columns");
  static constexpr int smem_bytes(int groups) {
    return 1024 + kStages * kStageBytes + kEpiBytes + kBarBytes + 2 * (groups + 1) * 4;
  }
};

struct alignas(64) Params {
  CUtensorMap tmA, tmB;     // operands
  CUtensorMap tmC, tmAux;   // outputs: bf16 box {64, 32}, or fp32 box {32, 32, 1} (kWeightGrad)
  const int* offsets;       // [groups + 1]
  int groups, rows;         // rows that exist
  int M, N, K;              // kWeightGrad: output [groups][M][N]; otherwise N output columns, K summed
  int band;                 // m tiles per raster band
  uint16_t* C;              // bf16 outputs, for the group's last rows
  int64_t ldc;
  uint16_t* aux_out;        // saved pre-activation (kBiasGelu)
  const uint16_t* aux;      // saved pre-activation (kGeluBwd)
  int64_t ld_aux;
  const uint16_t* bias;     // [groups][N] or null
  int accumulate;           // kWeightGrad: add to the output
  int* status;
};

struct alignas(8) Barriers {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint64_t tail_full;   // kWeightGrad: this CTA's loads of a partial step
  uint64_t tail_fixed;  // kWeightGrad: both CTAs have zeroed the foreign rows
  uint32_t tmem_base;
  int abort_flag;
  uint32_t peer_done;
  int bad_offsets;
};
static_assert(sizeof(Barriers) <= 256, "barrier slot");

struct Tile {
  int g;
  int m0, n0;       // first output row (kWeightGrad: inside the group's matrix) and column
  int row_end;      // kForward / kDataGrad: end of the group's rows
  int k0, kb;       // first summed row (kWeightGrad) and number of BK steps
  int tail;         // kWeightGrad: rows of the last step when it is partial, else 0
};

// Group table in shared memory: clamped offsets and first m tile of each group.
struct Table {
  const int* off;
  const int* first;
  int groups;
};

template <int CG, int BN, int OP>
__device__ __forceinline__ int tile_count(const Params& p, const Table& t) {
  using Cfg = Config<CG, BN>;
  const int nt = (p.N + BN - 1) / BN;
  if (OP == kWeightGrad) return p.groups * ((p.M + Cfg::kTileM - 1) / Cfg::kTileM) * nt;
  return t.first[t.groups] * nt;
}

template <int CG, int BN, int OP>
__device__ __forceinline__ Tile locate(const Params& p, const Table& t, int i) {
  using Cfg = Config<CG, BN>;
  const int nt = (p.N + BN - 1) / BN;
  Tile r;
  int mt, j;
  if (OP == kWeightGrad) {
    mt = (p.M + Cfg::kTileM - 1) / Cfg::kTileM;
    r.g = i / (mt * nt);
    j = i - r.g * mt * nt;
  } else {
    const int m = i / nt;
    int lo = 0, hi = t.groups - 1;  // the last group with first[g] <= m
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.first[mid] <= m) lo = mid; else hi = mid - 1;
    }
    r.g = lo;
    mt = t.first[lo + 1] - t.first[lo];
    j = i - t.first[lo] * nt;
  }
  // bands of p.band m tiles, m fastest: concurrent tiles share columns of W and a band of rows
  const int width = p.band * nt;
  const int band = j / width;
  const int size = min(mt - band * p.band, p.band);
  j -= band * width;
  r.m0 = (band * p.band + j % size) * Cfg::kTileM;
  r.n0 = j / size * BN;
  if (OP == kWeightGrad) {
    const int count = t.off[r.g + 1] - t.off[r.g];
    r.k0 = t.off[r.g];
    r.kb = (count + BK - 1) / BK;
    r.tail = count % BK;
    r.row_end = 0;
  } else {
    r.m0 += t.off[r.g];
    r.row_end = t.off[r.g + 1];
    r.k0 = 0;
    r.kb = (p.K + BK - 1) / BK;
    r.tail = 0;
  }
  return r;
}

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, uint32_t mbar_cluster, int x,
                                                 int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(mbar_cluster), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Bounded wait that also acquires what another CTA of the cluster released.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* status, int where) {
  const uint64_t start = globaltimer();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (globaltimer() - start > kWaitLimitNs) {
      record_status(status, kTimeoutPipeline, where);
      return false;
    }
  }
}

__device__ __forceinline__ void bulk_store_3d(const CUtensorMap* map, uint32_t buf, int x, int y, int z, bool add) {
  const uint64_t m = reinterpret_cast<uint64_t>(map);
  if (add)
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m),
        "r"(buf), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m),
                 "r"(buf), "r"(x), "r"(y), "r"(z)
                 : "memory");
}

// One epilogue warp's part of a tile: 32 accumulator rows x BN columns.
// MODE (gemm::EpiMode): kStore, kBias, kBiasGelu, kGeluBwd or kAccF32.
template <int BN, int MODE>
struct Epilogue {
  const Params& p;
  uint32_t base;  // this warp's two staging buffers
  int blocks = 0; // staged blocks so far
  static constexpr int kBuf = 4096;
  static constexpr bool kTwo = MODE == gemm::kBiasGelu;

  __device__ __forceinline__ void finish() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

  // The bulk store that last read the buffer about to be written is done with it.
  __device__ __forceinline__ void claim(int lane) {
    if (blocks >= (kTwo ? 1 : 2)) {
      if (lane == 0) {
        if (kTwo)
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        else
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      }
      __syncwarp();
    }
  }

  __device__ __forceinline__ static void row_copy(uint32_t buf, int lane, uint16_t* dst, int64_t ld, int rows, int col,
                                                  int N) {
    const int c = lane & 7;
    if (col + 8 * c >= N) return;
    for (int r = lane >> 3; r < rows; r += 4) {
      uint32_t a, b, d, e;
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(a), "=r"(b), "=r"(d), "=r"(e)
                   : "r"(buf + uint32_t(r * 128) + ((uint32_t(c) ^ uint32_t(r & 7)) << 4)));
      *reinterpret_cast<uint4*>(dst + int64_t(r) * ld + col + 8 * c) = make_uint4(a, b, d, e);
    }
  }

  // r: 32 fp32 accumulators of row `row` (this lane's), columns [col, col + 32).
  __device__ __forceinline__ void chunk_bf16(const Tile& t, int row, int col, int half, int valid,
                                             const uint32_t (&r)[32]) {
    const int lane = threadIdx.x & 31;
    float v[32], z[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
    if ((MODE == gemm::kBias || MODE == gemm::kBiasGelu) && p.bias) {
      const uint16_t* b = p.bias + int64_t(t.g) * p.N + col;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (col + 8 * q < p.N) {
          const uint4 w = __ldg(reinterpret_cast<const uint4*>(b + 8 * q));
          const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[8 * q + 2 * j] += __uint_as_float(a[j] << 16);
            v[8 * q + 2 * j + 1] += __uint_as_float(a[j] & 0xffff0000u);
          }
        }
      }
    }
    if (MODE == gemm::kBiasGelu) {
      // the activation is taken of the fp32 pre-activation; only its saved copy is rounded
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        z[j] = v[j];
        v[j] = gelu_erf(v[j]);
      }
    }
    if (MODE == gemm::kGeluBwd) {
      const uint16_t* a = p.aux + int64_t(row) * p.ld_aux + col;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (row < t.row_end && col + 8 * q < p.N) {
          const uint4 w = __ldg(reinterpret_cast<const uint4*>(a + 8 * q));
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[8 * q + 2 * j] *= gelu_erf_grad(__uint_as_float(u[j] << 16));
            v[8 * q + 2 * j + 1] *= gelu_erf_grad(__uint_as_float(u[j] & 0xffff0000u));
          }
        }
      }
    }
    const uint32_t buf = base + uint32_t((kTwo ? 0 : (blocks & 1)) * kBuf);
    const uint32_t bufz = base + uint32_t(kBuf);
    if (half == 0) claim(lane);
    gemm::TmaBf16Epi<gemm::kStore>::stage(buf, lane, half, v);
    if (kTwo) gemm::TmaBf16Epi<gemm::kStore>::stage(bufz, lane, half, z);
    if (half == 1) {
      const int col0 = col - 32, row0 = row - lane;
      if (valid >= 32) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          gemm::TmaBf16Epi<gemm::kStore>::store(&p.tmC, buf, col0, row0);
          if (kTwo) gemm::TmaBf16Epi<gemm::kStore>::store(&p.tmAux, bufz, col0, row0);
        }
      } else {  // the group's last rows: the rows after them belong to another group
        __syncwarp();
        row_copy(buf, lane, p.C + int64_t(row0) * p.ldc, p.ldc, valid, col0, p.N);
        if (kTwo) row_copy(bufz, lane, p.aux_out + int64_t(row0) * p.ld_aux, p.ld_aux, valid, col0, p.N);
        __syncwarp();
      }
      // one bulk group per staged block, also where it is empty, so that claim() counts blocks
      if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      ++blocks;
    }
  }

  __device__ __forceinline__ void chunk_f32(const Tile& t, int row, int col, bool zero, const uint32_t (&r)[32]) {
    const int lane = threadIdx.x & 31;
    const uint32_t buf = base + uint32_t((blocks & 1) * kBuf);
    claim(lane);
    const uint32_t rowa = buf + uint32_t(lane * 128), sw = uint32_t(lane & 7);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(rowa + ((uint32_t(c) ^ sw) << 4)),
                   "r"(zero ? 0u : r[4 * c]), "r"(zero ? 0u : r[4 * c + 1]), "r"(zero ? 0u : r[4 * c + 2]),
                   "r"(zero ? 0u : r[4 * c + 3])
                   : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      bulk_store_3d(&p.tmC, buf, col, row - lane, t.g, p.accumulate != 0);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    ++blocks;
  }
};

template <int CG, int BN, int OP, int MODE>
__device__ __forceinline__ void mainloop(const Params& p) {
  using Cfg = Config<CG, BN>;
  static_assert(CG == 1 || BN == 256, "SM pairs compute 256 x 256 tiles");
  constexpr int S = Cfg::kStages;
  constexpr bool kAMn = OP == kWeightGrad, kBMn = OP != kForward;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + S * Cfg::kStageBytes;
  Barriers* bars = reinterpret_cast<Barriers*>(epi_smem + Cfg::kEpiBytes);
  int* off = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + Cfg::kBarBytes);
  int* first = off + p.groups + 1;
  int* status = p.status;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? gemm2::cluster_ctarank() : 0u;
  const int unit = CG == 2 ? blockIdx.x >> 1 : blockIdx.x;
  const int units = CG == 2 ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->tmem_full[b], 1);
      mbar_init(&bars->tmem_empty[b], 4 * CG);
    }
    mbar_init(&bars->drain, 1);
    mbar_init(&bars->tail_full, 1);
    mbar_init(&bars->tail_fixed, CG);
    bars->abort_flag = 0;
    bars->peer_done = 0;
    fence_barrier_init();
    prefetch_tmap(&p.tmA);
    prefetch_tmap(&p.tmB);
  }
  if (warp == 1) {
    if (CG == 2) {
      gemm2::tmem_alloc2(&bars->tmem_base, Cfg::kTmemCols);
      gemm2::tmem_relinquish2();
    } else {
      tmem_alloc(&bars->tmem_base, Cfg::kTmemCols);
      tmem_relinquish();
    }
  }
  if (warp == 2) {
    // offsets must stay inside the existing rows and never decrease; a call
    // whose offsets do not is reported through the status word and computes nothing
    const int per = (p.groups + 31) / 32;
    bool bad = false;
    for (int i = lane; i <= p.groups; i += 32) {
      const int o = __ldg(p.offsets + i);
      const int c = max(0, min(o, p.rows));
      bad |= o != c;
      off[i] = c;
    }
    __syncwarp();
    int sum = 0;
    for (int i = 0; i < per; ++i) {
      const int g = lane * per + i;
      if (g < p.groups) {
        const int n = off[g + 1] - off[g];
        bad |= n < 0;
        sum += n > 0 ? (n + Cfg::kTileM - 1) / Cfg::kTileM : 0;
      }
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    int run = inc - sum;
    for (int i = 0; i < per; ++i) {
      const int g = lane * per + i;
      if (g < p.groups) {
        first[g] = run;
        const int n = off[g + 1] - off[g];
        run += n > 0 ? (n + Cfg::kTileM - 1) / Cfg::kTileM : 0;
      }
    }
    if (lane == 31) first[p.groups] = inc;
    if (bad) record_status(status, kBadArgument, 300, p.groups, p.rows);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) bars->bad_offsets = bad;
  }
  tc_fence_before();
  if (CG == 2)
    gemm2::cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  volatile int* abort_flag = &bars->abort_flag;
  const Table table{off, first, p.groups};
  // bad offsets: no tile is computed (both CTAs of a pair read the same offsets)
  const int tiles = bars->bad_offsets ? 0 : tile_count<CG, BN, OP>(p, table);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (OP == kWeightGrad || lane == 0) {
      uint32_t it = 0, tails = 0;
      bool ok = true;
      for (int i = unit; i < tiles && ok; i += units) {
        const Tile t = locate<CG, BN, OP>(p, table, i);
        if (OP == kWeightGrad && t.kb == 0 && p.accumulate) continue;
        const int m0 = t.m0 + int(rank) * 128, n0 = t.n0 + int(rank) * Cfg::kBRows;
        for (int kb = 0; kb < t.kb; ++kb, ++it) {
          const int s = it % S;
          bool go = mbar_wait(&bars->empty[s], ((it / S) & 1) ^ 1, status, 310) && !*abort_flag;
          if (OP == kWeightGrad) go = __all_sync(0xffffffffu, go);  // the whole warp runs this loop
          if (!go) { ok = false; *abort_flag = 1; break; }
          uint8_t* sa = smem + s * Cfg::kStageBytes;
          uint8_t* sb = sa + Cfg::kABytes;
          const bool partial = OP == kWeightGrad && t.tail != 0 && kb == t.kb - 1;
          const int k0 = t.k0 + kb * BK;
          if (lane == 0) {
            if (CG == 2 && !partial) {
              if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], 2 * Cfg::kStageBytes);
              const uint32_t fb = gemm2::mapa(smem_u32(&bars->full[s]), 0);
              if (!kAMn) {
                gemm2::tma_load_2d_pair(sa, &p.tmA, fb, k0, m0);
              } else {
                gemm2::tma_load_2d_pair(sa, &p.tmA, fb, m0, k0);
                gemm2::tma_load_2d_pair(sa + BK * 128, &p.tmA, fb, m0 + 64, k0);
              }
              if (OP == kForward) {
                tma_load_3d_pair(sb, &p.tmB, fb, k0, n0, t.g);
              } else if (OP == kDataGrad) {
                tma_load_3d_pair(sb, &p.tmB, fb, n0, k0, t.g);
                tma_load_3d_pair(sb + BK * 128, &p.tmB, fb, n0 + 64, k0, t.g);
              } else {
                gemm2::tma_load_2d_pair(sb, &p.tmB, fb, n0, k0);
                gemm2::tma_load_2d_pair(sb + BK * 128, &p.tmB, fb, n0 + 64, k0);
              }
            } else {
              uint64_t* bar = partial ? &bars->tail_full : &bars->full[s];
              mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
              if (!kAMn) {
                tma_load_2d(sa, &p.tmA, bar, k0, m0);
              } else {
                tma_load_2d(sa, &p.tmA, bar, m0, k0);
                tma_load_2d(sa + BK * 128, &p.tmA, bar, m0 + 64, k0);
              }
              if (OP == kForward) {
                tma_load_3d(sb, &p.tmB, bar, k0, n0, t.g);
              } else {
#pragma unroll
                for (int j = 0; j < Cfg::kBRows / 64; ++j) {
                  if (OP == kDataGrad)
                    tma_load_3d(sb + j * (BK * 128), &p.tmB, bar, n0 + 64 * j, k0, t.g);
                  else
                    tma_load_2d(sb + j * (BK * 128), &p.tmB, bar, n0 + 64 * j, k0);
                }
              }
            }
          }
          if (OP == kWeightGrad && partial) {
            // zeros over the rows of the next group, in both operands
            __syncwarp();
            const bool landed = mbar_wait(&bars->tail_full, tails & 1, status, 311);
            if (!__all_sync(0xffffffffu, landed)) { ok = false; *abort_flag = 1; break; }
            ++tails;
            constexpr int kBoxes = Cfg::kStageBytes / (BK * 128);
            const int lines = (BK - t.tail) * 8;  // 16-byte lines of the foreign rows of one box
            for (int j = lane; j < kBoxes * lines; j += 32) {
              const int box = j / lines, q = j - box * lines;
              *reinterpret_cast<uint4*>(sa + box * (BK * 128) + t.tail * 128 + q * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (CG == 2)
                gemm2::mbar_arrive_cluster(gemm2::mapa(smem_u32(&bars->tail_fixed), 0));
              else
                mbar_arrive(&bars->tail_fixed);
              if (rank == 0) mbar_arrive(&bars->full[s]);  // keeps the ring's phases
            }
          }
        }
        if (OP == kWeightGrad) __syncwarp();
      }
      if (!ok && rank == 0 && lane == 0) {
        // Drain: wait (bounded) for every stage that may still have bytes in flight.
        for (uint32_t j = (it >= S ? it - S : 0); j < it; ++j) mbar_wait(&bars->full[j % S], (j / S) & 1, status, 312);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_bf16(Cfg::kTileM, BN, kAMn, kBMn);
      uint32_t it = 0, tails = 0;
      int tc = 0;
      bool ok = true, issued = false;
      for (int i = unit; i < tiles && ok; i += units) {
        const Tile t = locate<CG, BN, OP>(p, table, i);
        if (OP == kWeightGrad && t.kb == 0 && p.accumulate) continue;
        const int b = tc & 1;
        if (!mbar_wait(&bars->tmem_empty[b], ((tc >> 1) & 1) ^ 1, status, 320)) { ok = false; *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t dcol = tmem_base + b * BN;
        for (int kb = 0; kb < t.kb; ++kb, ++it) {
          const int s = it % S;
          if (!mbar_wait(&bars->full[s], (it / S) & 1, status, 321)) { ok = false; *abort_flag = 1; break; }
          if (OP == kWeightGrad && t.tail != 0 && kb == t.kb - 1) {
            if (!mbar_wait_cluster(&bars->tail_fixed, tails & 1, status, 322)) { ok = false; *abort_flag = 1; break; }
            ++tails;
          }
          if (*abort_flag) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * Cfg::kStageBytes);
          const uint32_t sb = sa + Cfg::kABytes;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad = kAMn ? gemm::desc_mnmajor(sa + k * 16 * 128) : gemm::desc_kmajor(sa + k * 32);
            const uint64_t bd = kBMn ? gemm::desc_mnmajor(sb + k * 16 * 128) : gemm::desc_kmajor(sb + k * 32);
            if (CG == 2)
              gemm2::umma2_f16_ss(dcol, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
            else
              umma_f16_ss(dcol, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          issued = true;
          if (CG == 2)
            gemm2::umma2_commit_both(&bars->empty[s]);
          else
            umma_commit(&bars->empty[s]);
        }
        if (ok) {
          if (CG == 2)
            gemm2::umma2_commit_both(&bars->tmem_full[b]);
          else
            umma_commit(&bars->tmem_full[b]);
        }
        ++tc;
      }
      // Every MMA has landed before TMEM is released.
      if (issued) {
        if (CG == 2)
          gemm2::umma2_commit_both(&bars->drain);
        else
          umma_commit(&bars->drain);
        mbar_wait(&bars->drain, 0, status, 323);
      }
    }
  } else {
    // ---------------- Epilogue (warps 2..5) ----------------
    const int quarter = warp & 3;  // TMEM lanes [32*quarter, 32*quarter+32)
    Epilogue<BN, MODE> epi{p, smem_u32(epi_smem) + uint32_t(quarter * 2 * Cfg::kEpiBuf)};
    int tc = 0;
    for (int i = unit; i < tiles; i += units) {
      const Tile t = locate<CG, BN, OP>(p, table, i);
      if (OP == kWeightGrad && t.kb == 0 && p.accumulate) continue;
      const int b = tc & 1;
      bool ok = mbar_wait(&bars->tmem_full[b], (tc >> 1) & 1, status, 330);
      if (*abort_flag) ok = false;
      if (!ok) { *abort_flag = 1; break; }
      tc_fence_after();
      const int row0 = t.m0 + int(rank) * 128 + quarter * 32;
      const int valid = OP == kWeightGrad ? p.M - row0 : t.row_end - row0;
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem_base + (uint32_t(quarter * 32) << 16) + b * BN + c * 32, r);
        tmem_wait_ld();
        if (c == BN / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2)
              gemm2::mbar_arrive_cluster(gemm2::mapa(smem_u32(&bars->tmem_empty[b]), 0));
            else
              mbar_arrive(&bars->tmem_empty[b]);
          }
        }
        const int col = t.n0 + c * 32;
        if (valid <= 0) continue;
        if (OP == kWeightGrad) {
          if (col < p.N) epi.chunk_f32(t, row0 + lane, col, t.kb == 0, r);
        } else if (t.n0 + (c & ~1) * 32 < p.N) {
          epi.chunk_bf16(t, row0 + lane, col, c & 1, valid, r);
        }
      }
      ++tc;
    }
    epi.finish();
  }

  tc_fence_before();
  __syncthreads();
  if (CG == 2) {
    // Both CTAs have finished: a bounded handshake, then the paired TMEM free.
    if (threadIdx.x == 0) {
      gemm2::st_cluster_u32(gemm2::mapa(smem_u32(&bars->peer_done), rank ^ 1u), 1u);
      const uint64_t t0 = globaltimer();
      while (gemm2::ld_acquire_cta_u32(&bars->peer_done) == 0u) {
        if (globaltimer() - t0 > kWaitLimitNs) {
          record_status(status, kTimeoutLocal, 340);
          break;
        }
      }
    }
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) {
    if (CG == 2)
      gemm2::tmem_dealloc2(tmem_base, Cfg::kTmemCols);
    else
      tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

}  // namespace grouped
}  // namespace tdb
