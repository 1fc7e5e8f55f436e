// Microscaled 4-bit floating point ("MXFP4"): quantiser, its inverse and the
// product of two quantised operands on tcgen05 kind::mxf4.
//
// Values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two per
// byte with the even K index in the low half; each 32 consecutive K values of a
// row share a ue8m0 scale 2^(byte - 127).  For a block of absolute maximum a
// the exponent is the smallest e with a * 2^-e <= 6, so nothing saturates, and
// the scaled values round to nearest even.  A block that holds an infinity or
// NaN gets byte 255, which decodes as NaN; an all-zero block byte 0.
//
// Scales are stored in 512-byte atoms of 128 rows x 128 K values, byte
// (r % 32) * 16 + (r % 128) / 32 * 4 + j of row r and 32-value block j -- the
// order in which tcgen05.cp 32x128b.warpx4 brings them to TMEM.  Atoms of one
// 128-row block are consecutive along K, rounded up to an even number (a K
// step of the product is 256 values); blocks past K hold byte 0.  With
// offsets the rows of each group start a new block, so that a tile of the
// grouped product starts at a block wherever its group starts; when the groups
// hold at most 32 rows on average (block_rows) every 32 rows do, for tiles of
// 32 rows, and the other three quarters of their atoms stay unused.
#include <cuda_fp16.h>

#include "grouped_launch.cuh"

namespace tdb {
namespace mx4 {

using grouped::kMaxGroups;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;  // 256-value pieces of a row in flight per warp
constexpr int kMaxK = 65535 * kBatch * 256;  // 2^26 - 1024: a grid has at most 65535 blocks along K

// Block exponent from the bits of the largest |bf16|: the smallest e with
// a <= 6 * 2^e = 1.5 * 2^(e + 2), at least -127 (also for 0 and subnormals).
__host__ __device__ __forceinline__ int block_exponent(uint32_t abs_bits) {
  const int field = int(abs_bits >> 7);
  if (field == 0) return -127;
  const int e = field - 127 - 2 + ((abs_bits & 0x7f) > 0x40 ? 1 : 0);
  return e < -127 ? -127 : e;  // at most 126
}

__device__ __forceinline__ uint32_t max16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

__device__ __forceinline__ void e2m1x8_values(uint32_t q, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(q));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

struct Layout {
  const int* off;    // shared: group offsets, or null
  const int* block;  // shared: first block of each group
  int groups;
  int block_rows;        // 128, or 32 (with offsets)
  int rows, mat_blocks;  // without offsets: rows and blocks of one matrix
  // Scale block and row in it of row `r`; false for a row outside every group.
  __device__ __forceinline__ bool find(int r, int64_t& blk, int& in) const {
    if (!off) {
      const int m = r / rows;
      const int local = r - m * rows;
      blk = int64_t(m) * mat_blocks + local / 128;
      in = local % 128;
      return true;
    }
    if (r < off[0] || r >= off[groups]) return false;
    int lo = 0, hi = groups - 1;  // the last group that starts at or before r holds it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (off[mid] <= r) lo = mid; else hi = mid - 1;
    }
    const int local = r - off[lo];
    blk = block[lo] + local / block_rows;
    in = local % block_rows;
    return true;
  }
};

// Builds the layout's tables; returns false (status recorded) for bad offsets.
__device__ __forceinline__ bool make_layout(Layout& l, const int* offsets, int groups, int rows, int mat_blocks,
                                            int block_rows, int* sh, int* status) {
  l.off = nullptr;
  l.block = nullptr;
  l.groups = groups;
  l.block_rows = block_rows;
  l.rows = rows;
  l.mat_blocks = mat_blocks;
  if (!offsets) return true;
  int* off = sh;
  int* first = off + groups + 1;
  int* block = first + groups + 1;
  __shared__ int bad_offsets;
  if (threadIdx.x < 32) {
    const bool bad = grouped::load_offsets(offsets, groups, rows, off, status);
    __syncwarp();
    if (!bad) {
      if (block_rows == 32)
        grouped::scan_tiles<32, 32>(off, groups, first, block);
      else
        grouped::scan_tiles<128, 128>(off, groups, first, block);
    }
    if (threadIdx.x == 0) bad_offsets = bad;
  }
  __syncthreads();
  l.off = off;
  l.block = block;
  return !bad_offsets;
}

// A warp takes up to kBatch pieces of 256 consecutive values of a row (a pair
// of atoms' words each) at once, a lane 8 values of each.  Bound by the memory,
// as long as the instructions stay few: no division on the way (the row comes
// from the block, the pieces from its y), maxima on pairs.  4096 x 16384 in 32 us
// (5.3 TB/s; with divisions and single maxima 82 us).
__global__ void __launch_bounds__(kThreads) quantize_kernel(const uint16_t* __restrict__ x, int64_t ldx, int total_rows,
                                                            int K, uint8_t* __restrict__ q, uint8_t* __restrict__ sf,
                                                            const int* offsets, int groups, int rows, int mat_blocks, int block_rows,
                                                            int* status) {
  extern __shared__ int sh[];
  const int lane = threadIdx.x & 31;
  const int pieces = (K + 255) / 256;
  const int first = blockIdx.y * kBatch;
  const int k0 = first * 256 + lane * 8;
  auto load = [&](int64_t r, uint4 (&in)[kBatch]) {
    const uint16_t* src = x + r * ldx + k0;
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      in[b] = r < total_rows && k0 + b * 256 < K ? __ldg(reinterpret_cast<const uint4*>(src + b * 256))
                                                 : make_uint4(0, 0, 0, 0);
  };
  const int64_t step = int64_t(gridDim.x) * kWarps;
  int64_t r = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  uint4 in[kBatch];
  load(r, in);  // before the groups' table is built
  Layout l;
  if (!make_layout(l, offsets, groups, rows, mat_blocks, block_rows, sh, status)) return;
  for (; r < total_rows; r += step, load(r, in)) {
    int64_t blk;
    int row;
    if (!l.find(int(r), blk, row)) continue;
    uint8_t* dst = q + r * (K / 2) + k0 / 2;
    uint8_t* scale =
        sf + (blk * pieces + first) * 1024 + (lane >> 4) * 512 + (row & 31) * 16 + (row >> 5) * 4 + ((lane >> 2) & 3);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (first + b >= pieces) break;
      const uint32_t w[4] = {in[b].x, in[b].y, in[b].z, in[b].w};
      // largest |value| of the 32: as 16-bit integers the bits of |bf16| are ordered
      uint32_t pair = max16x2(max16x2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                              max16x2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
      pair = max16x2(pair, __shfl_xor_sync(0xffffffffu, pair, 1));
      pair = max16x2(pair, __shfl_xor_sync(0xffffffffu, pair, 2));
      const uint32_t top = max(pair & 0xffffu, pair >> 16);
      const bool finite = top < 0x7f80u;
      const int e = finite ? block_exponent(top) : 128;
      const float inv = __uint_as_float(uint32_t(127 - e) << 23);  // 2^-e, normal for e in [-127, 126]
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16) * inv;
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u) * inv;
      }
      if (k0 + b * 256 < K) *reinterpret_cast<uint32_t*>(dst + b * 128) = finite ? e2m1x8(v) : 0u;
      if ((lane & 3) == 0) scale[b * 1024] = uint8_t(e + 127);  // 0 past K
    }
  }
}

// The same walk backwards; 4096 x 16384 in 30 us (5.7 TB/s).
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf,
                                                              int total_rows, int K, uint16_t* __restrict__ out,
                                                              int64_t ldo, const int* offsets, int groups, int rows,
                                                              int mat_blocks, int block_rows, int* status) {
  extern __shared__ int sh[];
  Layout l;
  if (!make_layout(l, offsets, groups, rows, mat_blocks, block_rows, sh, status)) return;
  const int lane = threadIdx.x & 31;
  const int pieces = (K + 255) / 256;
  const int first = blockIdx.y * kBatch;
  for (int64_t r = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); r < total_rows; r += int64_t(gridDim.x) * kWarps) {
    int64_t blk;
    int row;
    if (!l.find(int(r), blk, row)) continue;
    const int k0 = first * 256 + lane * 8;
    const uint8_t* src = q + r * (K / 2) + k0 / 2;
    const uint8_t* scale = sf + (blk * pieces + first) * 1024 + (lane >> 4) * 512 + (row & 31) * 16 + (row >> 5) * 4 +
                           ((lane >> 2) & 3);
    uint32_t in[kBatch], byte[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const bool on = k0 + b * 256 < K;
      in[b] = on ? __ldg(reinterpret_cast<const uint32_t*>(src + b * 128)) : 0u;
      byte[b] = on ? __ldg(scale + b * 1024) : 0u;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (k0 + b * 256 >= K) break;
      const float s = __uint_as_float(byte[b] == 255u ? 0x7fffffffu : byte[b] == 0u ? 0x00400000u : byte[b] << 23);
      float v[8];
      e2m1x8_values(in[b], v);
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(v[2 * j] * s, v[2 * j + 1] * s);
      *reinterpret_cast<uint4*>(out + r * ldo + k0 + b * 256) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

static int64_t pairs_of(int64_t K) { return (K + 255) / 256; }

// Rows per scale block of an operand with offsets.
static int block_rows(int64_t rows, int64_t groups) { return groups > 0 && rows <= groups * 32 ? 32 : 128; }

// Scale blocks of an operand: matrices x ceil(rows / 128), or with groups the
// most that any offsets can need.
static int64_t blocks_of(int64_t matrices, int64_t rows, int64_t groups) {
  if (groups > 0) return rows / block_rows(rows, groups) + (rows < groups ? rows : groups);
  return matrices * ((rows + 127) / 128);
}

// With offsets every block builds the groups' table first: fewer, longer blocks.
static dim3 grid_for(int64_t rows, int64_t K, bool offsets) {
  const int64_t y = (pairs_of(K) + kBatch - 1) / kBatch;
  int64_t x = (rows + kWarps - 1) / kWarps;
  const int64_t most = int64_t(tdb_host::sm_count()) * 8 / y;
  if (offsets && x > most) x = most > 0 ? most : 1;
  return dim3(unsigned(x), unsigned(y));
}

static int check(const char* what, int64_t matrices, int64_t rows, int64_t K, int groups, const void* offsets) {
  if (matrices < 1 || rows < 0 || K < 32 || K % 32 || K > kMaxK || rows >= (int64_t(1) << 31) ||
      matrices >= (int64_t(1) << 31) || matrices * rows >= (int64_t(1) << 31) ||
      (offsets && (groups < 1 || groups > kMaxGroups || matrices != 1)))
    return tdb_host::fail(int(cudaErrorInvalidValue), "%s: K must be a multiple of 32, at most %d; 1..%d groups of one matrix's rows",
                          what, kMaxK, kMaxGroups);
  return 0;
}

}  // namespace mx4
}  // namespace tdb

using namespace tdb;

// Bytes of the scales of `matrices` [rows, K] operands, or (groups > 0) of one
// whose rows lie in that many groups.
TDB_API long long tdb_mx4_scale_bytes(long long matrices, long long rows, long long K, int groups) {
  return mx4::blocks_of(matrices, rows, groups) * mx4::pairs_of(K) * 1024;
}

// x bf16 [matrices * rows, K] (row stride ldx) -> q [matrices * rows, K / 2]
// (dense) and scales.
TDB_API int tdb_mx4_quantize(const void* x, int64_t ldx, int64_t matrices, int64_t rows, int64_t K, const int* offsets,
                             int groups, void* q, void* sf, void* stream) {
  if (int rc = mx4::check("mx4 quantize", matrices, rows, K, groups, offsets)) return rc;
  if (rows == 0) return 0;
  if (!x || !q || !sf || ldx % 8 || ldx < K || reinterpret_cast<uintptr_t>(x) % 16 ||
      (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(sf)) % 16)
    return tdb_host::fail(int(cudaErrorInvalidValue), "mx4 quantize: rows must be 16-byte aligned");
  mx4::quantize_kernel<<<mx4::grid_for(matrices * rows, K, offsets != nullptr), mx4::kThreads,
                         offsets ? size_t(3 * (groups + 1)) * 4 : 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint16_t*>(x), ldx, int(matrices * rows), int(K), static_cast<uint8_t*>(q), static_cast<uint8_t*>(sf),
      offsets, groups, int(rows), int((rows + 127) / 128), mx4::block_rows(rows, offsets ? groups : 0),
      tdb_host::status_ptr());
  tdb_host::launched(1);
  return int(cudaGetLastError());
}

// The bf16 values of a quantised operand (exact: three significant bits and a
// power of two), [matrices * rows, K] with row stride ldo.
TDB_API int tdb_mx4_dequantize(const void* q, const void* sf, int64_t matrices, int64_t rows, int64_t K,
                               const int* offsets, int groups, void* out, int64_t ldo, void* stream) {
  if (int rc = mx4::check("mx4 dequantize", matrices, rows, K, groups, offsets)) return rc;
  if (rows == 0) return 0;
  if (!out || !q || !sf || ldo % 8 || ldo < K || reinterpret_cast<uintptr_t>(out) % 16 ||
      (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(sf)) % 16)
    return tdb_host::fail(int(cudaErrorInvalidValue), "mx4 dequantize: rows must be 16-byte aligned");
  mx4::dequantize_kernel<<<mx4::grid_for(matrices * rows, K, offsets != nullptr), mx4::kThreads,
                           offsets ? size_t(3 * (groups + 1)) * 4 : 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(sf), int(matrices * rows), int(K), static_cast<uint16_t*>(out),
      ldo, offsets, groups, int(rows), int((rows + 127) / 128), mx4::block_rows(rows, offsets ? groups : 0),
      tdb_host::status_ptr());
  tdb_host::launched(1);
  return int(cudaGetLastError());
}

// Tile code that a 4-bit product takes (groups 0: without offsets).  32 where
// the scale blocks hold 32 rows, else as pick_rows_tile says, but not below 128
// (4096 rows x 16384 x 4096: 229 us with 128, 148 with 512; 512 x 4096 x 4096:
// 12.5 and 16.0).
TDB_API int tdb_mx4_pick_tile(long long rows, int groups, int N) {
  if (groups < 1) groups = 1;
  if (rows <= int64_t(groups) * 32) return 32;
  const int tile = tdb::grouped::pick_rows_tile(rows, groups, N, 0);
  return tile < 128 ? 128 : tile;
}

// C[r, :] = x[r] w_g^T (+ bias[g]) for the rows r of group g, x and w as
// tdb_mx4_quantize wrote them (x [rows, K] with the same offsets, w [groups, N,
// K] as `groups` matrices).  offsets null: one group of all rows (groups = 1).
TDB_API int tdb_mx4_gemm(const void* qx, const void* sfx, const void* qw, const void* sfw, const int* offsets, int groups,
                         void* C, int64_t ldc, int rows, int N, int K, const void* bias, int tile, void* stream) {
  using namespace tdb::grouped;
  if (groups < 1 || groups > kMaxGroups || (!offsets && groups != 1) || rows < 0 || N <= 0 || N % 8 || K < 32 ||
      K % 32 || K > mx4::kMaxK || rows > kMaxExtent || N > kMaxExtent)
    return tdb_host::fail(int(cudaErrorInvalidValue), "mx4 product: 1..%d groups, N a multiple of 8, K of 32 and at most %d",
                          kMaxGroups, mx4::kMaxK);
  if (rows == 0) return 0;
  if (!qx || !sfx || !qw || !sfw || !C || ldc % 8 || ldc < N ||
      (reinterpret_cast<uintptr_t>(qx) | reinterpret_cast<uintptr_t>(sfx) | reinterpret_cast<uintptr_t>(qw) |
       reinterpret_cast<uintptr_t>(sfw) | reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(bias)) % 16)
    return tdb_host::fail(int(cudaErrorInvalidValue), "mx4 product: operands must be 16-byte aligned, output rows too");
  if (tile == 0) tile = tdb_mx4_pick_tile(rows, offsets ? groups : 0, N);
  // tiles of 32 rows and scale blocks of 32 rows go together; up to 32 rows without offsets are one block either way
  const bool fits = offsets ? (tile == 32) == (mx4::block_rows(rows, groups) == 32) : tile != 32 || rows <= 32;
  if ((tile != 32 && tile != 128 && tile != 512) || !fits)
    return tdb_host::fail(int(cudaErrorInvalidValue), "mx4 product: tile must be 0, or one that fits the scale blocks: 32 "
                          "for at most 32 rows per group on average, else 128 or 512");
  const int64_t pairs = mx4::pairs_of(K);
  const int64_t x_blocks = offsets ? mx4::blocks_of(1, rows, groups) : mx4::blocks_of(1, rows, 0);
  const int64_t w_blocks = (N + 127) / 128;
  if (x_blocks * pairs >= (int64_t(1) << 31) || int64_t(groups) * w_blocks * pairs >= (int64_t(1) << 31))
    return tdb_host::fail(int(cudaErrorInvalidValue), "mx4 product: too many scale blocks");
  RowsParams p = {};
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
  int rc = tdb_host::make_tmap_3d(&p.tmA, qw, u8, 1, uint64_t(K / 2), uint64_t(N), uint64_t(groups), uint64_t(K / 2),
                                  uint64_t(K / 2) * uint64_t(N), 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = tdb_host::make_tmap_2d(&p.tmB, qx, u8, 1, uint64_t(K / 2), uint64_t(rows), uint64_t(K / 2), 128, tile == 512 ? 128 : 32,
                              CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = tdb_host::make_tmap_2d(&p.tmSfa, sfw, u32, 4, 256, uint64_t(int64_t(groups) * w_blocks * pairs), 256, 256, 1,
                              CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc) return rc;
  rc = tdb_host::make_tmap_2d(&p.tmSfb, sfx, u32, 4, 256, uint64_t(x_blocks * pairs), 256, 256, 1,
                              CU_TENSOR_MAP_SWIZZLE_NONE);
  if (rc) return rc;
  rc = make_output_map(&p.tmC, C, rows, N, ldc);
  if (rc) return rc;
  p.offsets = offsets;
  p.groups = groups;
  p.rows = rows;
  p.N = N;
  p.K = K;
  p.band = kBand;
  p.a_blocks = int(w_blocks);
  p.kpairs = int(pairs);
  p.C = static_cast<uint16_t*>(C);
  p.ldc = ldc;
  p.bias = static_cast<const uint16_t*>(bias);
  p.status = tdb_host::status_ptr();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tile == 512) return launch_rows<2, 256, kForward, gemm::kBias, true>(p, s);
  if (tile == 128) return launch_rows<1, 128, kForward, gemm::kBias, true>(p, s);
  return launch_rows<1, 32, kForward, gemm::kBias, true>(p, s);
}
