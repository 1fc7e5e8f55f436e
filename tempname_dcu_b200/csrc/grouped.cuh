// Grouped weight gradient: persistent warp-specialised tcgen05 GEMM whose summed
// dimension is ragged,
//
//   dW_g[n, k] = sum_{r in group g} dY[r, n] X[r, k]     (both MN-major)
//
// for the groups' rows [offsets[g], offsets[g+1]), read on the device.
//
// Partial steps.  The last step of a group whose size is not a multiple of 64
// holds rows of the next group.  The MMA issues only the K = 16 slices that
// have rows of the group; when the last slice is partial too, the step's loads
// complete on a barrier of their own CTA, and a warp writes zeros over the
// slice's foreign rows in both operands before the MMA may read it (a foreign
// row may hold NaN, so zeroing one operand would not do).  In the MN-major
// layout a row is a 128-byte line of each 64-column box, so the zeros need no
// swizzle.
//
// Sums.  The tensor core truncates when it adds to its fp32 accumulator, an
// error that grows with the number of additions and has one sign: 1170 rows
// were 2.2e-6 off (relative 2-norm), 8192 rows 4.4e-6, the output being fp32.
// So a chain of MMAs stops after kChain steps (512 rows) and the epilogue
// warps, which hold the output tile in registers, add the chain's result
// rounding to nearest: 4.8e-7 for any size.  Two TMEM accumulators alternate,
// so the MMAs do not wait; chains of 256 rows cost 7 % more time.
//
// Bounds: short sums the fp32 output (8 groups of 128 rows, 4096 x 4096: 108 us,
// 5 TB/s), long ones the rate of the steps.  7 groups, 4096 x 4096, from a cool
// start / back to back at the power limit (1.43 to 1.57 GHz at 990 W), us: 512
// rows each 134 / 154, 1024 228 / 253, 2048 399 / 449, 4096 760 / 862, 8192 1498 /
// 1706.  A group's row costs 26 ns (1.3 PFLOP/s cool, 1.14 at the limit), the
// output 25 to 55 us that the sums do not hide, the partial steps of 1170 rows
// some 18 us (272 / 303 in all).  Library products of the same operands with bf16
// outputs take 658 / 743 us for 4096 rows (1.46 and 1.30 PFLOP/s); the chains and
// the 256 x 256 tile's 64 KB of operands per step are what differs here.
//
// Few tiles with long sums (SPLIT, CG = 1): a cluster of CTAs computes one tile,
// each a part of the group's steps.  The tile's 16 boxes of 32 x 32 values go to
// the CTAs in turn; each leaves the boxes of the others in its shared memory and
// adds up its own, always in the same order: 2 groups of 4096 rows, 64 x 64,
// 26.2 us with one CTA each, 12.7 with eight; 2 of 8192, 512 x 512, 50 and 22;
// 4 of 1024, 256 x 1024 (two CTAs of 8 steps each), 10.4 and 10.5.
//
// The output leaves by TMA stores or, when adding, TMA reduce-adds (one writer
// per element: deterministic); an empty group's tiles are zeros, or skipped
// when adding.
//
// Warps: 0 TMA producer, 1 MMA issuer, 2 zeroes foreign rows, 3 reads the
// offsets, 4..11 epilogue (a quarter of the TMEM lanes and half of the columns
// each).  CG = 1: 128 x 128 tiles, CG = 2: 256 x 256 tiles on SM pairs with the
// barriers of gemm2.cuh.  All waits are bounded.
#pragma once
#include "grouped_rows.cuh"

namespace tdb {
namespace grouped {

constexpr int kWgThreads = 384;
// Registers per thread after the split, per warpgroup of 128 threads: the
// launch holds 384 x 168 = 64512, and 128 x 72 + 256 x 208 = 62464.
constexpr int kWgLightRegs = 72, kWgHeavyRegs = 208;
constexpr int kChain = 8;

template <int CG, int BN>
struct Config {
  static constexpr int kTileM = 128 * CG;      // output rows per tile (128 per CTA)
  static constexpr int kBRows = BN / CG;       // output columns whose operand this CTA stages
  static constexpr int kABytes = 128 * BK * 2;
  static constexpr int kBBytes = kBRows * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 5;
  static constexpr int kTmemCols = 2 * BN;     // two accumulators
  static constexpr int kWarpCols = BN / 2;     // output columns of an epilogue warp
  static constexpr int kBuf = 4096;            // 32 rows x 32 fp32 columns, one per epilogue warp
  static constexpr int kEpiBytes = 8 * kBuf;
  static constexpr int kBarBytes = 512;
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
  int parts;             // SPLIT: CTAs per tile
  int accumulate;
  int* status;
};

struct alignas(8) Barriers {
  uint64_t full[8];
  uint64_t empty[8];
  uint64_t part_full[8];   // this CTA's loads of a partial step, per stage
  uint64_t part_fixed[8];  // every CTA has zeroed its foreign rows, per stage
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  uint32_t peer_done;
  int bad_offsets;
};
static_assert(sizeof(Barriers) <= 512, "barrier slot");

struct Tile {
  int g;
  int m0, n0;   // first output row and column
  int k0, kb;   // first summed row and number of BK steps (SPLIT: of this CTA's part)
  int rows;     // of the group
  int last;     // rows of the last step, 1..64
  __device__ __forceinline__ bool patched() const { return (last & 15) != 0; }
};

template <int CG, int BN, bool SPLIT>
__device__ __forceinline__ Tile locate(const Params& p, const int* off, int i, int share) {
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
  r.last = count - (r.kb - 1) * BK;
  r.rows = count;
  if (SPLIT) {
    const int lo = int(int64_t(r.kb) * share / p.parts), hi = int(int64_t(r.kb) * (share + 1) / p.parts);
    if (hi != r.kb || lo == hi) r.last = BK;
    r.k0 += lo * BK;
    r.kb = hi - lo;
  }
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

template <int CG, int BN, bool SPLIT = false>
__device__ __forceinline__ void mainloop(const Params& p) {
  using Cfg = Config<CG, BN>;
  static_assert(!SPLIT || (CG == 1 && 16 * 4096 <= Cfg::kStages * Cfg::kStageBytes), "split sums");
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
  // SPLIT: a unit is a cluster of p.parts CTAs, and there are as many units as tiles
  const int share = SPLIT ? int(gemm2::cluster_ctarank()) : 0;
  const int unit = CG == 2 ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / p.parts : blockIdx.x;
  const int units = CG == 2 ? gridDim.x >> 1 : SPLIT ? gridDim.x / p.parts : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
      mbar_init(&bars->part_full[s], 1);
      mbar_init(&bars->part_fixed[s], CG);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->tmem_full[b], 1);
      mbar_init(&bars->tmem_empty[b], 8 * CG);
    }
    mbar_init(&bars->drain, 1);
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
  // everything above needs no memory of the kernels before this one
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 3) {
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
  const int tiles =
      bars->bad_offsets ? 0 : p.groups * ((p.M + Cfg::kTileM - 1) / Cfg::kTileM) * ((p.N + BN - 1) / BN);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWgLightRegs));
    if (warp == 0 && lane == 0) {
      // ---------------- TMA producer ----------------
      Ring<S> ring;
      uint32_t issued = 0, part = 0, partial = 0;  // per stage: phase bit of part_full, last use was partial
      bool ok = true;
      for (int i = unit; i < tiles && ok; i += units) {
        const Tile t = locate<CG, BN, SPLIT>(p, off, i, share);
        const int m0 = t.m0 + int(rank) * 128, n0 = t.n0 + int(rank) * Cfg::kBRows;
        int k0 = t.k0;
        for (int kb = 0; kb < t.kb; ++kb, k0 += BK, ring.next(), ++issued) {
          const int s = ring.s;
          if (!mbar_wait(&bars->empty[s], ring.phase ^ 1, status, 310)) {
            ok = false;
            *abort_flag = 1;
            break;
          }
          uint8_t* sa = smem + s * Cfg::kStageBytes;
          uint8_t* sb = sa + Cfg::kABytes;
          if (kb != t.kb - 1 || !t.patched()) {
            uint64_t* bar = &bars->full[s];
            partial &= ~(1u << s);
            if (rank == 0) mbar_arrive_expect_tx(bar, CG * Cfg::kStageBytes);
#pragma unroll
            for (int j = 0; j < 2; ++j) load_2d<CG>(sa + j * (BK * 128), &p.tmA, bar, m0 + 64 * j, k0);
#pragma unroll
            for (int j = 0; j < Cfg::kBRows / 64; ++j) load_2d<CG>(sb + j * (BK * 128), &p.tmB, bar, n0 + 64 * j, k0);
          } else {
            uint64_t* bar = &bars->part_full[s];
            partial |= 1u << s;
            part ^= 1u << s;
            mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
#pragma unroll
            for (int j = 0; j < 2; ++j) tma_load_2d(sa + j * (BK * 128), &p.tmA, bar, m0 + 64 * j, k0);
#pragma unroll
            for (int j = 0; j < Cfg::kBRows / 64; ++j) tma_load_2d(sb + j * (BK * 128), &p.tmB, bar, n0 + 64 * j, k0);
            if (rank == 0) mbar_arrive(&bars->full[s]);  // keeps the ring's phases; the MMA waits for part_fixed
          }
        }
      }
      if (!ok) {
        // Drain: wait (bounded) for every stage that may still have bytes in flight.
        if (rank == 0)
          for (uint32_t j = (issued >= S ? issued - S : 0); j < issued; ++j)
            mbar_wait(&bars->full[j % S], (j / S) & 1, status, 312);
        for (int s = 0; s < S; ++s)
          if ((partial >> s) & 1) mbar_wait(&bars->part_full[s], ((part >> s) & 1) ^ 1, status, 313);
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc = idesc_bf16(Cfg::kTileM, BN, true, true);
      Ring<S> ring;
      uint32_t part = 0;  // phase bit of each stage's part_fixed
      int tc = 0;         // chains
      bool ok = true, issued = false;
      const uint64_t a_desc = gemm::desc_mnmajor(smem_u32(smem));
      const uint64_t b_desc = gemm::desc_mnmajor(smem_u32(smem) + Cfg::kABytes);
      for (int i = unit; i < tiles && ok; i += units) {
        const Tile t = locate<CG, BN, SPLIT>(p, off, i, share);
        for (int c0 = 0; c0 < t.kb && ok; c0 += kChain, ++tc) {
          const int b = tc & 1, c1 = min(c0 + kChain, t.kb);
          if (!mbar_wait(&bars->tmem_empty[b], ((tc >> 1) & 1) ^ 1, status, 320)) { ok = false; break; }
          tc_fence_after();
          const uint32_t dcol = tmem_base + b * BN;
          for (int kb = c0; kb < c1; ++kb, ring.next()) {
            const int s = ring.s;
            if (!mbar_wait(&bars->full[s], ring.phase, status, 321)) { ok = false; break; }
            int slices = BK / 16;
            if (kb == t.kb - 1) {
              slices = (t.last + 15) >> 4;
              if (t.patched()) {
                if (!mbar_wait_cluster(&bars->part_fixed[s], (part >> s) & 1, status, 322)) { ok = false; break; }
                part ^= 1u << s;
              }
            }
            tc_fence_after();
            const uint64_t ad = a_desc + uint32_t(s * (Cfg::kStageBytes >> 4));
            const uint64_t bd = b_desc + uint32_t(s * (Cfg::kStageBytes >> 4));
            issue<CG>(dcol, ad, bd, idesc, kb != c0 ? 1u : 0u);
            if (slices == BK / 16) {
#pragma unroll
              for (int k = 1; k < BK / 16; ++k) issue<CG>(dcol, ad + k * 128, bd + k * 128, idesc, 1u);
            } else {
              for (int k = 1; k < slices; ++k) issue<CG>(dcol, ad + k * 128, bd + k * 128, idesc, 1u);
            }
            issued = true;
            commit<CG>(&bars->empty[s]);
          }
          if (ok) commit<CG>(&bars->tmem_full[b]);
        }
      }
      if (!ok) *abort_flag = 1;
      // Every MMA has landed before TMEM is released.
      if (issued) {
        commit<CG>(&bars->drain);
        mbar_wait(&bars->drain, 0, status, 323);
      }
    } else if (warp == 2) {
      // ---------------- Foreign rows ----------------
      uint32_t it = 0, part = 0;  // steps before and in this tile; phase bit of each stage's part_full
      for (int i = unit; i < tiles; i += units) {
        const Tile t = locate<CG, BN, SPLIT>(p, off, i, share);
        it += t.kb;
        if (t.kb == 0 || !t.patched()) continue;
        const int s = (it - 1) % S;
        bool go = mbar_wait(&bars->part_full[s], (part >> s) & 1, status, 311) && !*abort_flag;
        if (!__all_sync(0xffffffffu, go)) { *abort_flag = 1; break; }
        part ^= 1u << s;
        constexpr int kBoxes = Cfg::kStageBytes / (BK * 128);
        const int lines = (16 - (t.last & 15)) * 8;  // 16-byte lines of a box up to the slice's end
        uint8_t* from = smem + s * Cfg::kStageBytes + t.last * 128;
        for (int j = lane; j < lines; j += 32) {
#pragma unroll
          for (int box = 0; box < kBoxes; ++box)
            *reinterpret_cast<uint4*>(from + box * (BK * 128) + j * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_leader<CG>(&bars->part_fixed[s]);
      }
    }
  } else {
    // ---------------- Epilogue (warps 4..11) ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWgHeavyRegs));
    constexpr int kCols = Cfg::kWarpCols;
    const int quarter = warp & 3;  // TMEM lanes [32*quarter, 32*quarter+32)
    const int half = (warp - 4) >> 2;
    const uint32_t buf = smem_u32(epi_smem) + uint32_t((warp - 4) * Cfg::kBuf);
    int tc = 0;
    bool ok = true, joined = false;
    for (int i = unit; i < tiles && ok; i += units) {
      const Tile t = locate<CG, BN, SPLIT>(p, off, i, share);
      if (t.rows == 0 && p.accumulate) continue;
      float acc[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[j] = 0.f;
      for (int kb = 0; kb < t.kb; kb += kChain, ++tc) {
        const int b = tc & 1;
        ok = mbar_wait(&bars->tmem_full[b], (tc >> 1) & 1, status, 330);
        if (*abort_flag) ok = false;
        if (!ok) { *abort_flag = 1; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(tmem_base + (uint32_t(quarter * 32) << 16) + b * BN + half * kCols + c * 32, r);
          tmem_wait_ld();
          if (c == kCols / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_leader<CG>(&bars->tmem_empty[b]);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c * 32 + j] += __uint_as_float(r[j]);
        }
      }
      if (SPLIT) {
        // box q of the tile, column j of lane's row: 4 bytes per lane (the ring is free: its steps are summed)
        const uint32_t mine = smem_u32(smem) + uint32_t(lane * 4);
        const int q0 = (warp - 4) * (kCols / 32);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c)
            if ((q0 + c) % p.parts != share) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + uint32_t((q0 + c) * 4096 + j * 128)),
                             "f"(acc[c * 32 + j])
                             : "memory");
            }
        }
        cluster_barrier();
        joined = true;
        if (ok) {
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c)
            if ((q0 + c) % p.parts == share) {
              for (int o = 0; o < p.parts; ++o) {
                if (o == share) continue;
                const uint32_t from = gemm2::mapa(mine + uint32_t((q0 + c) * 4096), uint32_t(o));
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[c * 32 + j] += load_cluster(from + uint32_t(j * 128));
              }
            }
        }
      }
      if (!ok) break;
      const int row0 = t.m0 + int(rank) * 128 + quarter * 32;
      if (row0 >= p.M) continue;
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        const int col = t.n0 + half * kCols + c * 32;
        if (col < p.N && (!SPLIT || ((warp - 4) * (kCols / 32) + c) % p.parts == share)) {
          // the bulk store that last read the buffer is done with it
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
          const uint32_t rowa = buf + uint32_t(lane * 128), sw = uint32_t(lane & 7);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(rowa + ((uint32_t(k) ^ sw) << 4)),
                         "f"(acc[c * 32 + 4 * k]), "f"(acc[c * 32 + 4 * k + 1]), "f"(acc[c * 32 + 4 * k + 2]),
                         "f"(acc[c * 32 + 4 * k + 3])
                         : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            bulk_store_3d(&p.tmC, buf, col, row0, t.g, p.accumulate != 0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      }
    }
    if (SPLIT) {
      if (!joined) cluster_barrier();
      cluster_barrier();  // no CTA leaves while its sums are read
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  if (SPLIT && warp < 4) {  // the epilogue's two barriers
    cluster_barrier();
    cluster_barrier();
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
