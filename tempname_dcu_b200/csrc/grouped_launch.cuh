// Host side of the persistent grouped kernels: grid size and launch.
#pragma once
#include "grouped_rows.cuh"
#include "tensor_map.h"

namespace tdb {
namespace grouped {

constexpr int kBand = 8;  // token tiles per raster band

constexpr int kTwoPerSm = 113 * 1024;  // shared memory of a CTA when two share an SM

struct LaunchState {
  bool ready = false;
  int pairs = 0;  // SM pairs that can be resident at once (CG = 2)
};

// Launches `kern` on as many CTAs (CG = 1) or SM pairs (CG = 2) as there are
// tiles, at most one per SM of the caller's share.
template <int CG, class P>
static int launch_units(void (*kern)(P), const P& p, int threads, int64_t tiles, int smem, int max_smem, LaunchState* states,
                        cudaStream_t stream) {
  if (tiles >= (int64_t(1) << 31)) return tdb_host::fail(int(cudaErrorInvalidValue), "grouped: more than 2^31 output tiles");
  int dev = 0;
  cudaGetDevice(&dev);
  LaunchState& state = states[dev & 63];
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  // the setup of the kernel may run while the kernel before it on the stream ends
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  if (!state.ready) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem);
    if (e != cudaSuccess) return tdb_host::fail(int(e), "cudaFuncSetAttribute(grouped) failed");
    if (CG == 2) {
      cfg.gridDim = dim3(unsigned(tdb_host::sm_count() / 2 * 2));
      int n = 0;
      e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
      if (e != cudaSuccess || n <= 0) return tdb_host::fail(int(e), "grouped: no active SM pairs possible");
      state.pairs = n;
    }
    state.ready = true;
  }
  int64_t units = tdb_host::grid_sms() / CG;
  // two CTAs of the small tiles share an SM while the groups' table leaves them room and the caller has the whole GPU
  if (smem <= kTwoPerSm && tdb_host::grid_sms() == tdb_host::sm_count()) units *= 2;
  if (CG == 2 && units > state.pairs) units = state.pairs;
  if (units < 1) units = 1;
  if (tiles < units) units = tiles;
  cfg.gridDim = dim3(unsigned(units * CG));
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  tdb_host::launched(1);
  if (e != cudaSuccess) return tdb_host::fail(int(e), "grouped: launch failed");
  return 0;
}

constexpr int kSumSteps = 8;  // fewest steps of a sum that CTAs share

struct SplitState {
  bool ready = false;
  int clusters[9] = {};  // [CTAs per cluster]: clusters that can be resident at once, with one CTA per SM
};

// Launches `kern` with a cluster of CTAs on each tile, its p.parts set: as many
// as keep kSumSteps steps each while all tiles' clusters are resident.  Returns
// -1 if the tiles fill the SMs, the sums are too short or the caller has only a
// share of the SMs (clusters beyond it would not be resident).  Measured, bf16,
// microseconds with 1 / 2 / 4 / 8 CTAs: 4 tiles of 32 rows, 8192 summed values,
// 38.8 / 23.8 / 14.9 / 11.6; 66 tiles, 4096 values, 21.4 / 15.0 / 13.0 / 24.0
// (not all resident); 45 tiles of 128 rows, 8192 values, 51 / 31 / 39 / 48, with
// 3 25; 80 tiles of 32 rows, 512 values, 5.9 / 6.9.  4-bit, 40 rows of 1024 x
// 16384: 30 alone, 12.4 shared.
template <class P>
static int launch_split(void (*kern)(P), P p, int threads, int64_t tiles, int steps, int smem, int max_smem,
                        SplitState* states, cudaStream_t stream) {
  const int sms = tdb_host::sm_count();
  if (tiles < 1 || tiles * 5 > int64_t(sms) * 4 || steps < 2 * kSumSteps || tdb_host::grid_sms() != sms) return -1;
  int dev = 0;
  cudaGetDevice(&dev);
  SplitState& state = states[dev & 63];
  if (!state.ready) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem);
    if (e != cudaSuccess) return tdb_host::fail(int(e), "cudaFuncSetAttribute(grouped) failed");
    state.ready = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const int per_sm = smem <= kTwoPerSm ? 2 : 1;
  int parts = steps / kSumSteps < 8 ? steps / kSumSteps : 8;
  for (; parts > 1; --parts) {
    attr[0].val.clusterDim.x = unsigned(parts);
    int& clusters = state.clusters[parts];
    if (clusters == 0) {
      cfg.gridDim = dim3(unsigned(parts * sms));
      cfg.dynamicSmemBytes = size_t(max_smem);
      cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg);
      if (e != cudaSuccess) return tdb_host::fail(int(e), "grouped: cluster occupancy failed");
    }
    if (tiles <= clusters * per_sm) break;
  }
  if (parts < 2) return -1;
  p.parts = parts;
  cfg.gridDim = dim3(unsigned(tiles * parts));
  cfg.dynamicSmemBytes = size_t(smem);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  tdb_host::launched(1);
  if (e != cudaSuccess) return tdb_host::fail(int(e), "grouped: launch failed");
  return 0;
}

template <int CG, int BT, int OP, int MODE, bool MX4, bool SPLIT>
__global__ void __launch_bounds__(kThreads, BT == 32 ? 2 : 1) rows_kernel(const __grid_constant__ RowsParams p) {
  rows_mainloop<CG, BT, OP, MODE, MX4, SPLIT>(p);
}

template <int CG, int BT, int OP, int MODE, bool MX4>
static int launch_rows(const RowsParams& p, cudaStream_t stream) {
  using Cfg = RowsConfig<CG, BT, MX4>;
  static_assert(Cfg::smem_bytes(kMaxGroups) <= 227 * 1024, "shared memory budget");
  // most tiles that the rows can need: each group adds at most one partial tile
  const int64_t row_tiles = p.rows / BT + (p.rows < p.groups ? p.rows : p.groups);
  const int64_t tiles = row_tiles * ((p.N + Cfg::kTileN - 1) / Cfg::kTileN);
  if constexpr (CG == 1) {
    static SplitState state[64];
    const int steps = (p.K + (MX4 ? 255 : gemm::BK - 1)) / (MX4 ? 256 : gemm::BK);
    const int rc = launch_split(rows_kernel<CG, BT, OP, MODE, MX4, true>, p, kThreads, tiles, steps,
                                Cfg::smem_bytes(p.groups), Cfg::smem_bytes(kMaxGroups), state, stream);
    if (rc >= 0) return rc;
  }
  static LaunchState state[64];
  return launch_units<CG>(rows_kernel<CG, BT, OP, MODE, MX4, false>, p, kThreads, tiles, Cfg::smem_bytes(p.groups),
                          Cfg::smem_bytes(kMaxGroups), state, stream);
}

// Whether `tiles` CTAs' or pairs' worth of work fills at least half of `slots`.
static bool fills(int64_t tiles, int64_t slots) { return 2 * tiles >= slots; }

// Tile of a product of `rows` rows in `groups` groups with N output columns:
// 512 = up to 256 rows x 256 columns on SM pairs, 128 = 128 x 128, 32 = 32 x
// 128; the largest that an average group's rows nearly fill and that has tiles
// enough.  Measured with 8 groups, microseconds with 32 / 128 / 512: 4096 x 4096
// with 32 rows each 47 / 50 / 51, 96: 70 / 53 / 55, 128: 86 / 56 / 55, 160:
// 103 / 87 / 58, 384: 213 / 154 / 102; 512 x 2048, where large tiles leave SMs
// idle, with 64 rows each 13.1 / 14.3 / 14.8, 160: 13.8 / 15.4 / 17.0.  Tiles of
// 128 rows whose long sums CTAs share fill the SMs as well: 2 groups of 500 rows,
// 520 x 8192, 40 / 25; 300 rows of 1024 x 2048 in 2 groups, 11.0 / 10.6.
// Where CTAs cannot share them, SM pairs win long sums even when they fill less:
// 1024 x 2048 x 8192, 32 pairs, 54 / 43 with 128 / 512, with 2048 summed values
// 17.4 / 16.6, with 1024 10.7 / 12.1; 24 pairs 54 / 43.
static int pick_rows_tile(int64_t rows, int64_t groups, int N, int steps) {
  const int64_t used = rows < groups ? rows : groups;
  const int64_t average = used > 0 ? (rows + used - 1) / used : 0;
  const int sms = tdb_host::sm_count();
  const int64_t pairs = used * ((average + 255) / 256) * ((N + 255) / 256);
  const int64_t tiles = used * ((average + 127) / 128) * ((N + 127) / 128);
  if (average >= 128 && N >= 256 && (fills(pairs, sms / 2) || (steps >= 32 && tiles * 2 > sms))) return 512;
  const int shares = steps >= 32 ? (steps >= 128 ? 8 : steps / 16) : 1;
  if (average > 32 && fills(tiles * shares, sms)) return 128;
  return 32;
}

// bf16 output rows in blocks of 32 rows x 32 columns.
static int make_output_map(CUtensorMap* map, const void* C, int rows, int N, int64_t ldc) {
  return tdb_host::make_tmap_2d(map, C, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, uint64_t(N), uint64_t(rows), uint64_t(ldc),
                                32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

}  // namespace grouped
}  // namespace tdb
