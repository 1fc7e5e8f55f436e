// Entry points of the products grouped by expert (grouped.cuh) and the
// grouped bias gradient.
#include "grouped.cuh"
#include "grouped_few.cuh"
#include "grouped_launch.cuh"
#include "tensor_map.h"

namespace tdb {
namespace grouped {

template <int CG, int BN, bool SPLIT>
__global__ void __launch_bounds__(kWgThreads, 1) weight_grad_kernel(const __grid_constant__ Params p) {
  mainloop<CG, BN, SPLIT>(p);
}

template <int CG, int BN>
static int launch_weight_grad(const Params& p, cudaStream_t stream) {
  using Cfg = Config<CG, BN>;
  static_assert(Cfg::smem_bytes(kMaxGroups) <= 227 * 1024, "shared memory budget");
  const int64_t tiles = int64_t(p.groups) * ((p.M + Cfg::kTileM - 1) / Cfg::kTileM) * ((p.N + BN - 1) / BN);
  if constexpr (CG == 1) {
    static SplitState state[64];
    const int steps = p.rows / p.groups / gemm::BK;  // of an average group
    const int rc = launch_split(weight_grad_kernel<CG, BN, true>, p, kWgThreads, tiles, steps, Cfg::smem_bytes(p.groups),
                                Cfg::smem_bytes(kMaxGroups), state, stream);
    if (rc >= 0) return rc;
  }
  static LaunchState state[64];
  return launch_units<CG>(weight_grad_kernel<CG, BN, false>, p, kWgThreads, tiles, Cfg::smem_bytes(p.groups),
                          Cfg::smem_bytes(kMaxGroups), state, stream);
}

template <int OP, int MODE>
static int launch_rows_tile(int tile, const RowsParams& p, cudaStream_t s) {
  if (tile == 512) return launch_rows<2, 256, OP, MODE, false>(p, s);
  if (tile == 128) return launch_rows<1, 128, OP, MODE, false>(p, s);
  return launch_rows<1, 32, OP, MODE, false>(p, s);
}

// Bytes of the weights in use up to which the streaming kernel takes few rows: it
// starts sooner, the tiles read faster.
constexpr int64_t kFewBytes = 80 << 20;

// Tile of a call.  Forward with few rows: the streaming kernel (16) while the
// 128-column tiles of the groups that can have rows would leave SMs idle, also
// where CTAs share their sums, and the weights are at most kFewBytes.
// Microseconds with 16 / 32: one expert of 1024 x 1024 3.6 / 8.2, of 4096 x 4096
// (34 MB) 10.4 / 14.2, two (67 MB) 17.3 / 18.2; two of 2048 x 8192 (67 MB) 17.1 /
// 19.3, three (101 MB) 24.6 / 23.1; eight of 1024 x 8192 (134 MB) 31.0 / 27.3; two
// of 4096 x 16384 (268 MB) 54 / 49; of 16384 x 4096, 256 tiles, 52 / 46.  Weight
// gradient: SM pairs (512) when the sums are long enough to hide their larger
// tiles' output (8 groups of 4096 x 4096 with 256 rows each 126 us with 128, 137
// with 512; 384: 168 and 140; 1024: 374 and 249) and the tiles fill half of the
// pairs (8 of 512 x 512 with 1024 rows each: 11.5 and 14.0).
static int pick_tile(int op, int64_t rows, int groups, int M, int N) {
  if (op == kWeightGrad) {
    const int64_t tiles = int64_t(groups) * ((M + 255) / 256) * ((N + 255) / 256);
    return M >= 256 && N >= 256 && rows >= int64_t(groups) * 320 && fills(tiles, tdb_host::sm_count() / 2) ? 512 : 128;
  }
  if (op == kForward && rows <= kFewRows) {
    const int64_t used = rows < groups ? rows : groups, tiles = used * ((N + 127) / 128);
    if (tiles * 5 < int64_t(tdb_host::sm_count()) * 4 && used * N * M <= kFewBytes / 2) return 16;
  }
  return pick_rows_tile(rows, groups, N, (M + gemm::BK - 1) / gemm::BK);
}

template <int MODE>
static int launch_few(const RowsParams& p, const void* A, int64_t lda, const void* W, cudaStream_t s) {
  const int64_t units = int64_t((p.N + 15) / 16) * (p.rows < p.groups ? p.rows : p.groups);
  const int sms = tdb_host::grid_sms();
  const int64_t most = sms == tdb_host::sm_count() ? int64_t(sms) * 2 : sms;
  const unsigned grid = unsigned(units < most ? units : most);
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewRing);
    if (e != cudaSuccess) return tdb_host::fail(int(e), "cudaFuncSetAttribute(grouped few rows) failed");
    attr_set[dev & 63] = true;
  }
  few_rows_kernel<MODE><<<grid, kFewThreads, kFewRing, s>>>(
      static_cast<const uint16_t*>(A), lda, static_cast<const uint16_t*>(W), p.offsets, p.groups, p.rows, p.N, p.K, p.bias,
      p.C, p.ldc, p.aux_out, p.ld_aux, p.status);
  tdb_host::launched(1);
  return int(cudaGetLastError());
}

// Sums of dy's rows per group and column.  A block takes 64 columns of a group,
// 8 threads x 8 columns by 32 row lanes, joined in a fixed order.  PARTS > 1: a
// cluster of that many blocks shares a group's rows (each a contiguous part)
// and the first adds the others' sums, read from their shared memory; for
// outputs whose blocks would not fill the SMs.  Bound by reading dy: 8 groups,
// 8192 x 4096 in 6.3 us from L2 (10.2 us at the memory's copy rate).
template <int PARTS>
__global__ void __launch_bounds__(256) bias_grad_kernel(const uint16_t* __restrict__ dy, int64_t ld, int rows, int N,
                                                        const int* __restrict__ offsets, float* __restrict__ out,
                                                        int accumulate, int* status) {
  __shared__ float sh[32][65];
  __shared__ float sums[64];
  const int g = blockIdx.z, cx = threadIdx.x & 7, lane_row = threadIdx.x >> 3;
  const int col = blockIdx.y * 64 + cx * 8;
  const int first = offsets[g], last = offsets[g + 1];
  // Every block checks all offsets, so that none adds its sums to a call that
  // another one refuses: loaded beside the rows, compared where the threads meet
  // anyway.
  constexpr int kTurns = kMaxGroups / 256 + 1;
  int at[kTurns], before[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int e = i * 256 + int(threadIdx.x);
    const bool on = e <= int(gridDim.z);
    at[i] = on ? __ldg(offsets + e) : rows;
    before[i] = on && e ? __ldg(offsets + e - 1) : 0;
  }
  const bool own = first >= 0 && last >= first && last <= rows;  // else no row is read
  int lo = first, hi = last;
  if (PARTS > 1) {
    const int part = (last - first + PARTS - 1) / PARTS;
    lo = min(first + int(blockIdx.x) * part, last);
    hi = min(lo + part, last);
  }
  float acc[8] = {};
  if (own && col < N) {
#pragma unroll 4
    for (int r = lo + lane_row; r < hi; r += 32) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(dy + int64_t(r) * ld + col));
      const uint32_t a[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[2 * j] += __uint_as_float(a[j] << 16);
        acc[2 * j + 1] += __uint_as_float(a[j] & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[lane_row][cx * 8 + j] = acc[j];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) bad |= at[i] < before[i] || at[i] > rows;
  if (__syncthreads_or(bad)) {  // the same in every block
    if (threadIdx.x == 0) record_status(status, kBadArgument, 301, int(gridDim.z), rows);
    return;
  }
  float s = 0.f;
  if (threadIdx.x < 64) {
#pragma unroll
    for (int r = 0; r < 32; ++r) s += sh[r][threadIdx.x];
    if (PARTS > 1) sums[threadIdx.x] = s;
  }
  if (PARTS > 1) {
    gemm2::cluster_sync();
    if (blockIdx.x == 0 && threadIdx.x < 64) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(v)
                     : "r"(gemm2::mapa(smem_u32(&sums[threadIdx.x]), uint32_t(i)))
                     : "memory");
        s += v;
      }
    }
    gemm2::cluster_sync();  // no block leaves while its sums are read
    if (blockIdx.x != 0) return;
  }
  const int c = blockIdx.y * 64 + int(threadIdx.x);
  if (threadIdx.x < 64 && c < N) {
    float* o = out + int64_t(g) * N + c;
    *o = accumulate ? *o + s : s;
  }
}

template <int PARTS>
static int launch_bias_grad(const uint16_t* dY, int64_t ldy, int rows, int N, const int* offsets, int groups, float* out,
                            int accumulate, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PARTS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(PARTS, (N + 63) / 64, groups);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = PARTS > 1 ? 1 : 0;
  int* status = tdb_host::status_ptr();
  cudaError_t e = cudaLaunchKernelEx(&cfg, bias_grad_kernel<PARTS>, dY, ldy, rows, N, offsets, out, accumulate, status);
  tdb_host::launched(1);
  if (e != cudaSuccess) return tdb_host::fail(int(e), "grouped bias gradient: launch failed");
  return 0;
}

static bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

static int bad(const char* what) { return tdb_host::fail(int(cudaErrorInvalidValue), "%s", what); }

}  // namespace grouped
}  // namespace tdb

using namespace tdb;
using namespace tdb::grouped;

// Tile code that a grouped call takes (op 0 forward, 1 data gradient: M summed
// values; 2 weight gradient: M x N outputs); see pick_tile.
TDB_API int tdb_grouped_pick_tile(int op, long long rows, int groups, int M, int N) {
  return tdb::grouped::pick_tile(op, rows, groups, M, N);
}

// C[r, :] = epilogue(A[r, :] W_g) for the rows r of group g, g = 0..groups:
//   data_grad 0: A [rows, K], W [groups, N, K], C [rows, N] = A W_g^T (+ bias)
//   data_grad 1: A [rows, K], W [groups, K, N], C [rows, N] = A W_g
// mode kStore, kBias, kBiasGelu (data_grad 0; aux_out gets the pre-activation)
// or kGeluBwd (data_grad 1; aux holds it).  Rows outside every group keep
// their contents.  tile 0 picks the tile.
TDB_API int tdb_grouped_gemm(const void* A, int64_t lda, const void* W, int data_grad, const int* offsets, int groups,
                             void* C, int64_t ldc, int rows, int N, int K, int mode, const void* bias, const void* aux,
                             int64_t ld_aux, void* aux_out, int tile, void* stream) {
  if (groups < 1 || groups > kMaxGroups || rows < 0 || N <= 0 || K <= 0 || N % 8 || K % 8 || rows > kMaxExtent ||
      N > kMaxExtent || K > kMaxExtent)
    return tdb_host::fail(int(cudaErrorInvalidValue), "grouped: 1..%d groups, N and K multiples of 8, extents below 2^31 - 1024",
                          kMaxGroups);
  if (rows == 0) return 0;
  if (!A || !W || !C || !offsets || lda % 8 || lda < K || ldc % 8 || ldc < N || misaligned(A) || misaligned(W) ||
      misaligned(C) || (bias && misaligned(bias)))
    return bad("grouped: operands must be 16-byte aligned with 16-byte row strides");
  const bool modes_ok = data_grad ? (mode == gemm::kStore || mode == gemm::kGeluBwd)
                                  : (mode == gemm::kStore || mode == gemm::kBias || mode == gemm::kBiasGelu);
  if (!modes_ok || (mode == gemm::kBias && !bias)) return bad("grouped: epilogue mode not available");
  if ((mode == gemm::kBiasGelu && (!aux_out || misaligned(aux_out) || ld_aux % 8 || ld_aux < N)) ||
      (mode == gemm::kGeluBwd && (!aux || misaligned(aux) || ld_aux % 8 || ld_aux < N)))
    return bad("grouped: the pre-activation must be 16-byte aligned with 16-byte row strides");
  if (tile == 0) tile = tdb::grouped::pick_tile(data_grad ? kDataGrad : kForward, rows, groups, K, N);
  if (tile != 32 && tile != 128 && tile != 512 && (tile != 16 || data_grad || rows > kFewRows || N > (1 << 26)))
    return bad("grouped: tile must be 0, 32, 128 or 512 (16: forward with at most 16 rows and 2^26 columns)");
  RowsParams p = {};
  p.offsets = offsets;
  p.groups = groups;
  p.rows = rows;
  p.N = N;
  p.K = K;
  p.band = kBand;
  p.C = static_cast<uint16_t*>(C);
  p.ldc = ldc;
  p.aux_out = static_cast<uint16_t*>(aux_out);
  p.aux = static_cast<const uint16_t*>(aux);
  p.ld_aux = ld_aux;
  p.bias = static_cast<const uint16_t*>(bias);
  p.status = tdb_host::status_ptr();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tile == 16)
    return mode == gemm::kBiasGelu ? launch_few<gemm::kBiasGelu>(p, A, lda, W, s) : launch_few<gemm::kBias>(p, A, lda, W, s);
  const uint32_t box_rows = tile == 512 ? 128 : 32;
  int rc = tdb_host::make_tmap_2d(&p.tmB, A, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, uint64_t(K), uint64_t(rows),
                                  uint64_t(lda), gemm::BK, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  if (data_grad)
    rc = tdb_host::make_tmap_3d(&p.tmA, W, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, uint64_t(N), uint64_t(K),
                                uint64_t(groups), uint64_t(N), uint64_t(N) * uint64_t(K), 64, gemm::BK,
                                CU_TENSOR_MAP_SWIZZLE_128B);
  else
    rc = tdb_host::make_tmap_3d(&p.tmA, W, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, uint64_t(K), uint64_t(N),
                                uint64_t(groups), uint64_t(K), uint64_t(N) * uint64_t(K), gemm::BK, 128,
                                CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = make_output_map(&p.tmC, C, rows, N, ldc);
  if (rc) return rc;
  if (mode == gemm::kBiasGelu) {
    rc = make_output_map(&p.tmAux, aux_out, rows, N, ld_aux);
    if (rc) return rc;
  }
  if (data_grad)
    return mode == gemm::kGeluBwd ? launch_rows_tile<kDataGrad, gemm::kGeluBwd>(tile, p, s)
                                  : launch_rows_tile<kDataGrad, gemm::kStore>(tile, p, s);
  if (mode == gemm::kBiasGelu) return launch_rows_tile<kForward, gemm::kBiasGelu>(tile, p, s);
  if (mode == gemm::kBias) return launch_rows_tile<kForward, gemm::kBias>(tile, p, s);
  return launch_rows_tile<kForward, gemm::kStore>(tile, p, s);
}

// C[g] (fp32 [groups, N, K]) (+)= dY_g^T X_g over the rows of group g:
// dY [rows, N], X [rows, K].
TDB_API int tdb_grouped_weight_grad(const void* dY, int64_t ldy, const void* X, int64_t ldx, const int* offsets,
                                    int groups, float* C, int rows, int N, int K, int accumulate, int tile,
                                    void* stream) {
  if (groups < 1 || groups > kMaxGroups || rows < 0 || N <= 0 || K <= 0 || N % 8 || K % 8 || rows > kMaxExtent ||
      N > kMaxExtent || K > kMaxExtent)
    return tdb_host::fail(int(cudaErrorInvalidValue),
                          "grouped weight gradient: 1..%d groups, N and K multiples of 8, extents below 2^31 - 1024",
                          kMaxGroups);
  if (!C || misaligned(C)) return bad("grouped weight gradient: the output must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (accumulate) return 0;
    return int(cudaMemsetAsync(C, 0, size_t(groups) * N * K * sizeof(float), s));
  }
  if (!dY || !X || !offsets || ldy % 8 || ldy < N || ldx % 8 || ldx < K || misaligned(dY) || misaligned(X))
    return bad("grouped weight gradient: operands must be 16-byte aligned with 16-byte row strides");
  if (tile == 0) tile = tdb::grouped::pick_tile(kWeightGrad, rows, groups, N, K);
  if (tile != 128 && tile != 512) return bad("grouped weight gradient: tile must be 0, 128 or 512");
  Params p = {};
  int rc = tdb_host::make_tmap_2d(&p.tmA, dY, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, uint64_t(N), uint64_t(rows),
                                  uint64_t(ldy), 64, gemm::BK, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = tdb_host::make_tmap_2d(&p.tmB, X, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, uint64_t(K), uint64_t(rows),
                              uint64_t(ldx), 64, gemm::BK, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = tdb_host::make_tmap_3d(&p.tmC, C, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, uint64_t(K), uint64_t(N), uint64_t(groups),
                              uint64_t(K), uint64_t(N) * uint64_t(K), 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  p.offsets = offsets;
  p.groups = groups;
  p.rows = rows;
  p.M = N;
  p.N = K;
  p.band = 8;
  p.accumulate = accumulate;
  p.status = tdb_host::status_ptr();
  return tile == 512 ? launch_weight_grad<2, 256>(p, s) : launch_weight_grad<1, 128>(p, s);
}

// out[g] (fp32 [groups, N]) (+)= the sum of dY's rows of group g.
TDB_API int tdb_grouped_bias_grad(const void* dY, int64_t ldy, const int* offsets, int groups, float* out, int rows,
                                  int N, int accumulate, void* stream) {
  if (groups < 1 || groups > kMaxGroups || rows < 0 || N <= 0 || N % 8 || rows > kMaxExtent || N > kMaxExtent)
    return tdb_host::fail(int(cudaErrorInvalidValue), "grouped bias gradient: 1..%d groups, N a multiple of 8", kMaxGroups);
  if (!out || !offsets || (rows > 0 && (!dY || ldy % 8 || ldy < N || misaligned(dY))))
    return bad("grouped bias gradient: rows must be 16-byte aligned");
  if ((N + 63) / 64 > 65535) return bad("grouped bias gradient: at most 65535 x 64 columns");
  const uint16_t* dy = static_cast<const uint16_t*>(dY);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // eight blocks per group and 64 columns unless the groups' own blocks fill the SMs (8 of 256 threads each)
  if (int64_t(groups) * ((N + 63) / 64) >= int64_t(tdb_host::sm_count()) * 2)
    return launch_bias_grad<1>(dy, ldy, rows, N, offsets, groups, out, accumulate, s);
  return launch_bias_grad<8>(dy, ldy, rows, N, offsets, groups, out, accumulate, s);
}
