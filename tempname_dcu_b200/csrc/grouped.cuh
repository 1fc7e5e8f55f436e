// Grouped weight gradient: persistent warp-specialised tcgen05 GEMM whose summed
// dimension is ragged,
//
//   dW_g[n, k] = sum_{r in group g} dY[r, n] X[r, k]     (both MN-major)
//
// for the groups' rows [offsets[g], offsets[g+1]), read on the device.  The
// last 64-row step of a group whose size is not a multiple of 64 is fetched
// apart (onto a barrier of this CTA), and the producer warp writes zeros over
// the next group's rows of both operands before the MMA may read the step: a
// foreign row may hold NaN, so zeroing one operand would not do.  In the
// MN-major layout a row is a 128-byte line of each 64-column box, so the zeros
// need no swizzle.  The fp32 output leaves by TMA stores or, when adding, TMA
// reduce-adds (one writer per element: deterministic); an empty group's tiles
// are zeros, or skipped when adding.
//
// Roles and barriers are those of gemm.cuh (CG = 1: 128 x 128 tiles) and
// gemm2.cuh (CG = 2: 256 x 256 tiles on SM pairs): warp 0 TMA producer, warp 1
// MMA issuer, warps 2..5 epilogue; all waits are bounded.
#pragma once
#include "grouped_rows.cuh"

namespace tdb {
namespace grouped {

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
    return 1024 + kStages * kStageBytes + kEpiBytes + kBarBytes + (groups + 1) * 4;
  }
};

struct alignas(64) Params {
  CUtensorMap tmA, tmB;  // dY, X: boxes of 64 rows x 64 columns
  CUtensorMap tmC;       // output, fp32 box {32, 32, 1}
  const int* offsets;    // [groups + 1]
  int groups, rows;
  int M, N;              // output [groups][M][N]
  int band;              // m tiles per raster band
  int accumulate;
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
  int m0, n0;   // first output row and column
  int k0, kb;   // first summed row and number of BK steps
  int tail;     // rows of the last step when it is partial, else 0
};

template <int CG, int BN>
__device__ __forceinline__ Tile locate(const Params& p, const int* off, int i) {
  using Cfg = Config<CG, BN>;
  const int nt = (p.N + BN - 1) / BN, mt = (p.M + Cfg::kTileM - 1) / Cfg::kTileM;
  Tile r;
  r.g = i / (mt * nt);
  int j = i - r.g * mt * nt;
  const int width = p.band * nt;
  const int band = j / width;
  const int size = min(mt - band * p.band, p.band);
  j -= band * width;
  r.m0 = (band * p.band + j % size) * Cfg::kTileM;
  r.n0 = j / size * BN;
  const int count = off[r.g + 1] - off[r.g];
  r.k0 = off[r.g];
  r.kb = (count + BK - 1) / BK;
  r.tail = count % BK;
  return r;
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

template <int CG, int BN>
__device__ __forceinline__ void mainloop(const Params& p) {
  using Cfg = Config<CG, BN>;
  static_assert(CG == 1 || BN == 256, "SM pairs compute 256 x 256 tiles");
  constexpr int S = Cfg::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + S * Cfg::kStageBytes;
  Barriers* bars = reinterpret_cast<Barriers*>(epi_smem + Cfg::kEpiBytes);
  int* off = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + Cfg::kBarBytes);
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
    const bool bad = load_offsets(p.offsets, p.groups, p.rows, off, status);
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
  // bad offsets: no tile is computed (both CTAs of a pair read the same offsets)
  const int tiles = bars->bad_offsets ? 0 : p.groups * ((p.M + Cfg::kTileM - 1) / Cfg::kTileM) * ((p.N + BN - 1) / BN);

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    {  // the whole warp runs this loop (it zeroes foreign rows), lane 0 issues the loads
      uint32_t it = 0, tails = 0;
      bool ok = true;
      for (int i = unit; i < tiles && ok; i += units) {
        const Tile t = locate<CG, BN>(p, off, i);
        if (t.kb == 0 && p.accumulate) continue;
        const int m0 = t.m0 + int(rank) * 128, n0 = t.n0 + int(rank) * Cfg::kBRows;
        for (int kb = 0; kb < t.kb; ++kb, ++it) {
          const int s = it % S;
          bool go = mbar_wait(&bars->empty[s], ((it / S) & 1) ^ 1, status, 310) && !*abort_flag;
          go = __all_sync(0xffffffffu, go);
          if (!go) { ok = false; *abort_flag = 1; break; }
          uint8_t* sa = smem + s * Cfg::kStageBytes;
          uint8_t* sb = sa + Cfg::kABytes;
          const bool partial = t.tail != 0 && kb == t.kb - 1;
          const int k0 = t.k0 + kb * BK;
          if (lane == 0) {
            if (!partial) {
              uint64_t* bar = &bars->full[s];
              if (rank == 0) mbar_arrive_expect_tx(bar, CG * Cfg::kStageBytes);
#pragma unroll
              for (int j = 0; j < 2; ++j) load_2d<CG>(sa + j * (BK * 128), &p.tmA, bar, m0 + 64 * j, k0);
#pragma unroll
              for (int j = 0; j < Cfg::kBRows / 64; ++j) load_2d<CG>(sb + j * (BK * 128), &p.tmB, bar, n0 + 64 * j, k0);
            } else {
              uint64_t* bar = &bars->tail_full;
              mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
#pragma unroll
              for (int j = 0; j < 2; ++j) tma_load_2d(sa + j * (BK * 128), &p.tmA, bar, m0 + 64 * j, k0);
#pragma unroll
              for (int j = 0; j < Cfg::kBRows / 64; ++j) tma_load_2d(sb + j * (BK * 128), &p.tmB, bar, n0 + 64 * j, k0);
            }
          }
          if (partial) {
            // zeros over the rows of the next group, in both operands
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
              arrive_leader<CG>(&bars->tail_fixed);
              if (rank == 0) mbar_arrive(&bars->full[s]);  // keeps the ring's phases
            }
          }
        }
      }
      if (!ok && rank == 0 && lane == 0) {
        // Drain: wait (bounded) for every stage that may still have bytes in flight.
        for (uint32_t j = (it >= S ? it - S : 0); j < it; ++j) mbar_wait(&bars->full[j % S], (j / S) & 1, status, 312);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_bf16(Cfg::kTileM, BN, true, true);
      uint32_t it = 0, tails = 0;
      int tc = 0;
      bool ok = true, issued = false;
      for (int i = unit; i < tiles && ok; i += units) {
        const Tile t = locate<CG, BN>(p, off, i);
        if (t.kb == 0 && p.accumulate) continue;
        const int b = tc & 1;
        if (!mbar_wait(&bars->tmem_empty[b], ((tc >> 1) & 1) ^ 1, status, 320)) { ok = false; *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t dcol = tmem_base + b * BN;
        for (int kb = 0; kb < t.kb; ++kb, ++it) {
          const int s = it % S;
          if (!mbar_wait(&bars->full[s], (it / S) & 1, status, 321)) { ok = false; *abort_flag = 1; break; }
          if (t.tail != 0 && kb == t.kb - 1) {
            if (!mbar_wait_cluster(&bars->tail_fixed, tails & 1, status, 322)) { ok = false; *abort_flag = 1; break; }
            ++tails;
          }
          if (*abort_flag) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * Cfg::kStageBytes);
          const uint32_t sb = sa + Cfg::kABytes;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad = gemm::desc_mnmajor(sa + k * 16 * 128);
            const uint64_t bd = gemm::desc_mnmajor(sb + k * 16 * 128);
            if (CG == 2)
              gemm2::umma2_f16_ss(dcol, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
            else
              umma_f16_ss(dcol, ad, bd, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          issued = true;
          commit<CG>(&bars->empty[s]);
        }
        if (ok) commit<CG>(&bars->tmem_full[b]);
        ++tc;
      }
      // Every MMA has landed before TMEM is released.
      if (issued) {
        commit<CG>(&bars->drain);
        mbar_wait(&bars->drain, 0, status, 323);
      }
    }
  } else {
    // ---------------- Epilogue (warps 2..5) ----------------
    const int quarter = warp & 3;  // TMEM lanes [32*quarter, 32*quarter+32)
    const uint32_t base = smem_u32(epi_smem) + uint32_t(quarter * 2 * Cfg::kEpiBuf);
    int tc = 0, staged = 0;
    for (int i = unit; i < tiles; i += units) {
      const Tile t = locate<CG, BN>(p, off, i);
      if (t.kb == 0 && p.accumulate) continue;
      const int b = tc & 1;
      bool ok = mbar_wait(&bars->tmem_full[b], (tc >> 1) & 1, status, 330);
      if (*abort_flag) ok = false;
      if (!ok) { *abort_flag = 1; break; }
      tc_fence_after();
      const int row0 = t.m0 + int(rank) * 128 + quarter * 32;
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem_base + (uint32_t(quarter * 32) << 16) + b * BN + c * 32, r);
        tmem_wait_ld();
        if (c == BN / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_leader<CG>(&bars->tmem_empty[b]);
        }
        const int col = t.n0 + c * 32;
        if (row0 >= p.M || col >= p.N) continue;
        const uint32_t buf = base + uint32_t((staged & 1) * Cfg::kEpiBuf);
        if (staged >= 2) {  // the bulk store that last read the buffer is done with it
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
        }
        const uint32_t rowa = buf + uint32_t(lane * 128), sw = uint32_t(lane & 7);
        const bool zero = t.kb == 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(rowa + ((uint32_t(k) ^ sw) << 4)),
                       "r"(zero ? 0u : r[4 * k]), "r"(zero ? 0u : r[4 * k + 1]), "r"(zero ? 0u : r[4 * k + 2]),
                       "r"(zero ? 0u : r[4 * k + 3])
                       : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          bulk_store_3d(&p.tmC, buf, col, row0, t.g, p.accumulate != 0);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        ++staged;
      }
      ++tc;
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
