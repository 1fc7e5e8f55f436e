// Grouped forward and data-gradient products (and the 4-bit forward product)
// with the weights on the M side of the tensor-core tile:
//
//   kForward   Y[r, n]  = sum_k W_g[n, k] X[r, k]     (W K-major,  X K-major)
//   kDataGrad  dX[r, k] = sum_n W_g[n, k] dY[r, n]    (W MN-major, dY K-major)
//
// A tile is 128*CG output columns (weight rows) by up to BT rows of one group.
// The ragged dimension is the N of tcgen05.mma, which may be any multiple of
// 16, so a group's rows are rounded up to 16 and not to a whole tile; a
// group's rows are split evenly over its tiles.  With 8 groups of 512 rows on
// average, 256-row tiles on the M side spend a fifth of the multiplications on
// rows that do not exist.
//
// Bounds: with few rows the reading of the weights (two CTAs per SM with four
// stages each keep the memory busy: one token through two experts of 16384 x
// 4096 in 47 us, 5.7 TB/s), with many the tensor cores and, back to back, the
// power limit (8 groups of 512 rows through 16384 x 4096: 460 us, 1.2 PFLOP/s
// sustained, against 467 us for eight library products; 8 uneven groups with
// GELU and both outputs 585 us, the data gradient with GELU' 590 us).  A step is
// fetched by two requests: 64-row boxes (three requests) took 6 to 10 % longer.
//
// The accumulator then holds output columns along TMEM lanes and rows along
// TMEM columns.  The epilogue reads it with tcgen05.ld 16x256b, whose register
// layout is that of 8x8 fragments, works on it elementwise and transposes
// with stmatrix.trans into row-major blocks of 32 rows x 32 columns (64-byte
// rows, 64-byte swizzle), which leave by TMA; blocks with fewer rows (the end
// of a group) leave row by row, so rows of other groups are never written.
//
// MX4 (kForward): both operands hold e2m1 values, two per byte, with ue8m0
// scales per 32 K values in 512-byte atoms (128 rows x 128 K values, the byte
// order of MxOperands in gemm.cuh); a K step is 256 values (128 bytes) and two
// atoms per 128 rows.  The scales of the weight rows are loaded by the CTA
// that owns the rows, those of the token rows by both CTAs of a pair.  Large
// products are bound by what L2 delivers to the SMs (35 KB per CTA and step)
// and by the scales' copies: 4096 x 16384 x 4096 in 148 us (3.7 PFLOP/s), 8192^3
// in 256 us (4.3 PFLOP/s); without either scale loads or copies, as an
// experiment, 205 us.  64 rows over 16 experts of 4096 x 4096: 27 us, 5.2 TB/s.
//
// Roles as in gemm.cuh: warp 0 TMA producer, warp 1 MMA issuer, warps 2..5
// epilogue; CG = 2 runs on SM pairs.  All waits are bounded.
#pragma once
#include "gemm.cuh"
#include "gemm2.cuh"
#include "gemm_epi.cuh"

namespace tdb {
namespace grouped {

using gemm::BK;
constexpr int kThreads = 192;
constexpr int kMaxGroups = 1024;
constexpr int kMaxExtent = 0x7fffffff - 1024;  // rows and columns: tile coordinates past the end stay 32-bit

enum Op : int { kForward = 0, kDataGrad = 1, kWeightGrad = 2 };

template <int CG, int BT, bool MX4>
struct RowsConfig {
  static constexpr int kTileN = 128 * CG;              // output columns per tile
  static constexpr int kBRows = BT / CG;               // token rows staged per CTA
  static constexpr int kBox = CG == 2 ? 128 : 32;      // token rows per TMA copy: only boxes with rows are loaded
  static constexpr int kABytes = 128 * 128;            // 128 rows of 64 bf16 or 256 e2m1
  static constexpr int kBBytes = kBRows * 128;
  static constexpr int kBlockRows = BT == 32 ? 32 : 128;  // token rows that a scale block holds (see mx4.cu)
  static constexpr int kBlocksB = BT / kBlockRows;        // scale blocks of a tile's token rows
  static constexpr int kSfBytes = MX4 ? 1024 * (1 + kBlocksB) : 0;
  static constexpr int kStageBytes = kABytes + kBBytes + kSfBytes;
  static constexpr int kStages = BT == 32 ? 4 : (MX4 ? 5 : 6);
  static constexpr int kAccums = MX4 && BT == 256 ? 1 : 2;  // beside two of 256 columns no scale would fit
  static constexpr int kSfCols = MX4 ? 8 * (1 + kBlocksB) : 0;
  static constexpr int kUsedCols = kAccums * BT + kStages * kSfCols;
  static constexpr int kTmemCols = kUsedCols <= 64 ? 64 : kUsedCols <= 128 ? 128 : kUsedCols <= 256 ? 256 : 512;
  static_assert(kUsedCols <= 512, "TMEM columns");
  static constexpr int kBuf = 2048;                    // 32 rows x 32 bf16 columns
  static constexpr int kEpiBytes = 4 * 2 * kBuf;
  static constexpr int kBarBytes = 512;
  static constexpr int smem_bytes(int groups) {
    return 1024 + kStages * kStageBytes + kEpiBytes + kBarBytes + 3 * (groups + 1) * 4;
  }
};

struct alignas(64) RowsParams {
  CUtensorMap tmA, tmB;      // weights (3-D), token rows (2-D)
  CUtensorMap tmSfa, tmSfb;  // MX4: pairs of scale atoms (rows of 256 words)
  CUtensorMap tmC, tmAux;    // outputs: box {32, 32}, 64-byte swizzle
  const int* offsets;        // [groups + 1], or null: one group of all rows
  int groups, rows;
  int N, K;                  // output columns, summed values
  int parts;                 // SPLIT: CTAs per tile
  int band;                  // token tiles per raster band
  int a_blocks, kpairs;      // MX4: 128-row blocks of a weight matrix, atom pairs along K
  uint16_t* C;
  int64_t ldc;
  uint16_t* aux_out;         // saved pre-activation (kBiasGelu)
  const uint16_t* aux;       // saved pre-activation (kGeluBwd)
  int64_t ld_aux;
  const uint16_t* bias;      // [groups][N] or null
  int* status;
};

struct alignas(8) RowsBarriers {
  uint64_t full[16];
  uint64_t empty[16];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  uint32_t peer_done;
  int bad_offsets;
};
static_assert(sizeof(RowsBarriers) <= 512, "barrier slot");

struct RowsTile {
  int g;
  int n0;            // first output column of the tile (the pair's)
  int r0, count;     // first row and number of rows
  int block;         // MX4: first scale block of the rows
  int mma_n;         // count rounded up to 16
};

// The groups' table in shared memory: row offsets, first tile and (MX4) first
// scale block of each group.
struct RowsTable {
  const int* off;
  const int* first;
  const int* block;
};

// Tiles of a group: ceil(n / BT) of them, of equal size up to 16 rows (MX4: of
// BT rows, since tiles start where scale blocks do).
template <int BT, bool MX4>
__device__ __forceinline__ int rows_per_tile(int n, int tiles) {
  if (MX4) return BT;
  const int even = (n + tiles - 1) / tiles;
  return (even + 15) & ~15;
}

// Reads and checks the offsets (one warp).  Offsets must stay inside the
// existing rows and never decrease; otherwise the call computes nothing and
// says so in the status word.
__device__ __forceinline__ bool load_offsets(const int* offsets, int groups, int rows, int* off, int* status) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  int last = 0;  // of the entries before this stride
  for (int i0 = 0; i0 <= groups; i0 += 32) {
    const int i = i0 + lane;
    const int o = i > groups ? rows : offsets ? __ldg(offsets + i) : (i ? rows : 0);
    int before = __shfl_up_sync(0xffffffffu, o, 1);
    if (lane == 0) before = last;
    bad |= o < before || o > rows;
    if (i <= groups) off[i] = o;
    last = __shfl_sync(0xffffffffu, o, 31);
  }
  if (bad) record_status(status, kBadArgument, 300, groups, rows);
  return __any_sync(0xffffffffu, bad);
}

// First tile of BT rows (and first scale block of BR rows, BR > 0) of each
// group, by one warp.
template <int BT, int BR>
__device__ __forceinline__ void scan_tiles(const int* off, int groups, int* first, int* block) {
  constexpr bool BLOCKS = BR > 0;
  constexpr int kRows = BLOCKS ? BR : 1;
  const int lane = threadIdx.x & 31;
  const int per = (groups + 31) / 32;
  int sum = 0, bsum = 0;
  for (int g = lane * per; g < min(lane * per + per, groups); ++g) {
    const int n = off[g + 1] - off[g];
    sum += (n + BT - 1) / BT;
    bsum += (n + kRows - 1) / kRows;
  }
  int inc = sum, binc = bsum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    const int bup = __shfl_up_sync(0xffffffffu, binc, o);
    if (lane >= o) {
      inc += up;
      binc += bup;
    }
  }
  int run = inc - sum, brun = binc - bsum;
  for (int g = lane * per; g < min(lane * per + per, groups); ++g) {
    const int n = off[g + 1] - off[g];
    first[g] = run;
    run += (n + BT - 1) / BT;
    if (BLOCKS) {
      block[g] = brun;
      brun += (n + kRows - 1) / kRows;
    }
  }
  if (lane == 31) first[groups] = inc;
}

template <int CG, int BT, bool MX4>
__device__ __forceinline__ RowsTile rows_locate(const RowsParams& p, const RowsTable& t, int i) {
  constexpr int kTileN = RowsConfig<CG, BT, MX4>::kTileN;
  const int nt = (p.N + kTileN - 1) / kTileN;
  const int m = i / nt;
  int lo = 0, hi = p.groups - 1;  // the last group with first[g] <= m
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= m) lo = mid; else hi = mid - 1;
  }
  RowsTile r;
  r.g = lo;
  const int mt = t.first[lo + 1] - t.first[lo];
  int j = i - t.first[lo] * nt;
  // bands of p.band token tiles, token tiles fastest: concurrent tiles share weights and a band of rows
  const int width = p.band * nt;
  const int band = j / width;
  const int size = min(mt - band * p.band, p.band);
  j -= band * width;
  const int mi = band * p.band + j % size;
  r.n0 = j / size * kTileN;
  const int n = t.off[lo + 1] - t.off[lo];
  const int step = rows_per_tile<BT, MX4>(n, mt);
  r.r0 = t.off[lo] + mi * step;
  r.count = min(step, n - mi * step);  // > 0: (mt - 1) * step <= (mt - 1) * BT < n
  r.block = MX4 ? t.block[lo] + mi * RowsConfig<CG, BT, MX4>::kBlocksB : 0;
  r.mma_n = (r.count + 15) & ~15;
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

// Position in the ring of S stages.  The issuing threads have a few hundred
// cycles per step, so it is stepped, not divided.
template <int S>
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++s == S) {
      s = 0;
      phase ^= 1;
    }
  }
};

template <int CG>
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  if (CG == 2)
    gemm2::tma_load_2d_pair(dst, map, gemm2::mapa(smem_u32(bar), 0), x, y);
  else
    tma_load_2d(dst, map, bar, x, y);
}
template <int CG>
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  if (CG == 2)
    tma_load_3d_pair(dst, map, gemm2::mapa(smem_u32(bar), 0), x, y, z);
  else
    tma_load_3d(dst, map, bar, x, y, z);
}
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (CG == 2)
    gemm2::umma2_commit_both(bar);
  else
    umma_commit(bar);
}
template <int CG>
__device__ __forceinline__ void issue(uint32_t tmem_d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (CG == 2)
    gemm2::umma2_f16_ss(tmem_d, ad, bd, idesc, accumulate);
  else
    umma_f16_ss(tmem_d, ad, bd, idesc, accumulate);
}
template <int CG>
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  if (CG == 2)
    gemm2::mbar_arrive_cluster(gemm2::mapa(smem_u32(bar), 0));
  else
    mbar_arrive(bar);
}

// Instruction descriptor of kind::mxf4: e2m1 A and B (format 1), ue8m0 scales
// (bit 23), dense K = 64 (bit 31 = 0); [4,6) and [29,31) the scale ids of B, A.
__device__ __forceinline__ uint32_t idesc_mxf4(int m, int n) {
  return (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 4) << 24);
}

// One K = 64 step; sf_byte 0 or 2 picks the pair of scale bytes of the column word.
template <int CG>
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t sfa_col, uint32_t sfb_col, uint32_t sf_byte, uint32_t accumulate) {
  const uint32_t id = idesc | (sf_byte << 29) | (sf_byte << 4);
  const uint32_t ta = sfa_col | (sf_byte << 30), tb = sfb_col | (sf_byte << 30);
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(id), "r"(accumulate), "r"(ta), "r"(tb));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(id), "r"(accumulate), "r"(ta), "r"(tb));
}

// 512-byte scale atom -> 4 TMEM columns (CG = 2: in each CTA from its own shared memory).
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = smem_desc_plain(saddr, 0, 128);
  if (CG == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    tmem_cp_32x128b_x4(taddr, desc);
}

// 16 TMEM lanes x 32 columns: 8x8 fragments, f[4i + 2h + e] = row 8h + lane/4,
// column 8i + 2(lane%4) + e.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// GELU and its derivative with the normal distribution function from Abramowitz
// and Stegun's approximation 7.1.26 of erfc (|error| < 1.5e-7): with z = |x| /
// sqrt 2, t = 1 / (1 + 0.3275911 z),
//   erfc(z) = t (a1 + t (a2 + t (a3 + t (a4 + t a5)))) exp(-z^2),
// whose exponential is the density's too.  Half of it is the probability above
// |x|, so gelu(x) = max(x, 0) - |x| tail and gelu'(x) = 1 - v (x >= 0) or v (x <
// 0) with v = tail - |x| density; nothing cancels where the results are small.
// What is left is the formula's own error: below 1.5e-7 / 2 (times |x| for gelu)
// anywhere, 5e-4 of gelu(x) at -4, 2.5e-3 at -5.5 (half a bf16 step is 2e-3 to
// 4e-3), 3 % at -12, where gelu is 1e-32; an |x|^2 th part of that in gelu'(x).
// Some 14 instructions each.  At the power limit the epilogue's instructions are
// paid for in the tensor cores' clock: 4096 rows through 16384 x 4096 with GELU
// 463 -> 452 us against the form with a division, a selection and separate factors.
// |x| is cut at 1e30, since an infinity times its tail of 0 would be NaN; a NaN
// stays one through the exponential.
__device__ __forceinline__ float gelu_density(float x) {  // exp(-x^2 / 2)
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-0.72134752f * x * x));
  return e;
}
__device__ __forceinline__ float gelu_tail(float z) {  // the probability above z over gelu_density(z)
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f * 0.70710678f, z, 1.f)));
  float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = fmaf(t, q, 0.5f * 1.421413741f);
  q = fmaf(t, q, 0.5f * -0.284496736f);
  q = fmaf(t, q, 0.5f * 0.254829592f);
  return t * q;
}
__device__ __forceinline__ float gelu(float x) {
  const float z = fminf(fabsf(x), 1e30f);
  return fmaf(-z, gelu_tail(z) * gelu_density(x), fmaxf(x, 0.f));
}
__device__ __forceinline__ float gelu_slope(float x) {
  const float z = fminf(fabsf(x), 1e30f);
  const float v = fmaf(-0.3989422804f, z, gelu_tail(z)) * gelu_density(x);
  return x >= 0.f ? 1.f - v : v;
}

// One epilogue warp: 32 output columns (TMEM lanes) of a tile, 32 rows at a
// time.  MODE (gemm::EpiMode): kStore, kBias, kBiasGelu or kGeluBwd.
template <int MODE>
struct RowsEpilogue {
  const RowsParams& p;
  uint32_t base;    // this warp's two staging buffers
  int blocks = 0;   // staged blocks so far
  float bias[4] = {0.f, 0.f, 0.f, 0.f};  // of columns 8h + lane/4
  static constexpr int kBuf = 2048;
  static constexpr bool kTwo = MODE == gemm::kBiasGelu;

  __device__ __forceinline__ void finish() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

  // 16-byte piece `c` of staged row `row` (64-byte rows, 64-byte swizzle).
  __device__ __forceinline__ static uint32_t piece(uint32_t buf, int row, int c) {
    return buf + uint32_t(row * 64) + (uint32_t(c ^ ((row >> 1) & 3)) << 4);
  }

  __device__ __forceinline__ void tile_begin(const RowsTile& t, int col0) {
    if ((MODE == gemm::kBias || MODE == gemm::kBiasGelu) && p.bias) {
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int col = col0 + 8 * h + (lane >> 2);
        bias[h] = col < p.N ? bf16_bits_to_float(__ldg(p.bias + int64_t(t.g) * p.N + col)) : 0.f;
      }
    }
  }

  // The saved pre-activations of one block (four 16-byte pieces per lane).
  __device__ __forceinline__ void load_aux(int row0, int valid, int col0, uint4 (&a)[4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2), c = lane & 3;
      a[i] = make_uint4(0, 0, 0, 0);
      if (r < valid && col0 + 8 * c < p.N)
        a[i] = __ldg(reinterpret_cast<const uint4*>(p.aux + int64_t(row0 + r) * p.ld_aux + col0) + c);
    }
  }

  // bf16 fragments of a block: w[4i + m] holds rows 8i + 2(lane%4) + {0, 1} of column 8m + lane/4.
  __device__ __forceinline__ static void pack(const float (&v)[32], uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[4 * i] = pack_bf16x2(v[4 * i], v[4 * i + 1]);
      w[4 * i + 1] = pack_bf16x2(v[4 * i + 2], v[4 * i + 3]);
      w[4 * i + 2] = pack_bf16x2(v[16 + 4 * i], v[16 + 4 * i + 1]);
      w[4 * i + 3] = pack_bf16x2(v[16 + 4 * i + 2], v[16 + 4 * i + 3]);
    }
  }
  __device__ __forceinline__ static void stage(uint32_t buf, const uint32_t (&w)[16]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // rows 8i .. 8i+7
      stmatrix_x4_trans(piece(buf, 8 * i + (lane & 7), lane >> 3), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }

  __device__ __forceinline__ void copy_rows(uint32_t buf, uint16_t* dst, int64_t ld, int rows, int col0) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    if (col0 + 8 * c >= p.N) return;
    for (int r = lane >> 2; r < rows; r += 8) {
      uint32_t x, y, z, w;
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(x), "=r"(y), "=r"(z), "=r"(w)
                   : "r"(piece(buf, r, c)));
      *reinterpret_cast<uint4*>(dst + int64_t(r) * ld + col0 + 8 * c) = make_uint4(x, y, z, w);
    }
  }

  // The bulk store that last read the buffer about to be written is done with it.
  __device__ __forceinline__ uint32_t claim() {
    if (blocks >= (kTwo ? 1 : 2)) {
      if ((threadIdx.x & 31) == 0) {
        if (kTwo)
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        else
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      }
      __syncwarp();
    }
    return base + uint32_t((kTwo ? 0 : (blocks & 1)) * kBuf);
  }

  // Writes the staged block (kTwo: and the pre-activations staged behind it),
  // `valid` (<= 32 used) rows from row0.
  __device__ __forceinline__ void release(uint32_t buf, int row0, int valid, int col0) {
    const int lane = threadIdx.x & 31;
    if (valid >= 32) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        gemm::TmaBf16Epi<gemm::kStore>::store(&p.tmC, buf, col0, row0);
        if (kTwo) gemm::TmaBf16Epi<gemm::kStore>::store(&p.tmAux, base + uint32_t(kBuf), col0, row0);
      }
    } else {  // the group's last rows: those after them belong to another group
      __syncwarp();
      copy_rows(buf, p.C + int64_t(row0) * p.ldc, p.ldc, valid, col0);
      if (kTwo) copy_rows(base + uint32_t(kBuf), p.aux_out + int64_t(row0) * p.ld_aux, p.ld_aux, valid, col0);
      __syncwarp();
    }
    // one bulk group per block, also where it is empty, so that claim() counts blocks
    if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    ++blocks;
  }

  __device__ __forceinline__ void add_bias(float (&v)[32]) const {
    if (MODE == gemm::kBias || MODE == gemm::kBiasGelu) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += bias[2 * (j >> 4) + ((j >> 1) & 1)];
    }
  }

  // v[16h' + 4i + 2h + e]: column 16h' + 8h + lane/4, row 8i + 2(lane%4) + e of
  // the block of `valid` (<= 32 used) rows at row0.
  __device__ __forceinline__ void block(float (&v)[32], const uint4 (&a)[4], int row0, int valid, int col0) {
    const int lane = threadIdx.x & 31;
    const uint32_t buf = claim();
    uint32_t w[16];
    add_bias(v);
    if (MODE == gemm::kBiasGelu) {
      // the activation is taken of the fp32 pre-activation; only its saved copy is rounded
      pack(v, w);
      stage(base + uint32_t(kBuf), w);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = gelu(v[j]);
    }
    if (MODE == gemm::kGeluBwd) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(piece(buf, 8 * i + (lane >> 2), lane & 3)),
                     "r"(a[i].x), "r"(a[i].y), "r"(a[i].z), "r"(a[i].w)
                     : "memory");
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t z[4];  // columns 8m + lane/4, rows 8i + 2(lane%4) + {0, 1}
        ldmatrix_x4_trans(piece(buf, 8 * i + (lane & 7), lane >> 3), z);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int j = 16 * (m >> 1) + 4 * i + 2 * (m & 1);
          v[j] *= gelu_slope(__uint_as_float(z[m] << 16));
          v[j + 1] *= gelu_slope(__uint_as_float(z[m] & 0xffff0000u));
        }
      }
      __syncwarp();
    }
    pack(v, w);
    stage(buf, w);
    release(buf, row0, valid, col0);
  }
};

// A barrier over the cluster's threads, for warps whose lanes took different ways.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// SPLIT (CG = 1): a cluster of CTAs computes one tile, each a part of the summed
// steps.  They leave their accumulators in shared memory; chunk c (32 rows) is
// then added up, always in the same order, and stored by CTA c % parts.  For
// long sums whose tiles are few.
template <int CG, int BT, int OP, int MODE, bool MX4, bool SPLIT = false>
__device__ __forceinline__ void rows_mainloop(const RowsParams& p) {
  using Cfg = RowsConfig<CG, BT, MX4>;
  static_assert(!SPLIT || (CG == 1 && Cfg::kAccums == 2 && BT * 512 <= Cfg::kStages * Cfg::kStageBytes), "split sums");
  constexpr int S = Cfg::kStages;
  constexpr bool kAMn = OP == kDataGrad;
  constexpr int kStep = MX4 ? 256 : BK;  // summed values per stage
  static_assert(!MX4 || OP == kForward, "4-bit operands are K-major");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + S * Cfg::kStageBytes;
  RowsBarriers* bars = reinterpret_cast<RowsBarriers*>(epi_smem + Cfg::kEpiBytes);
  int* off = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + Cfg::kBarBytes);
  int* first = off + p.groups + 1;
  int* block = first + p.groups + 1;
  int* status = p.status;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? gemm2::cluster_ctarank() : 0u;
  // SPLIT: a unit is a cluster of `parts` CTAs, and there are as many units as tiles
  const int part = SPLIT ? int(gemm2::cluster_ctarank()) : 0, parts = SPLIT ? p.parts : 1;
  const int unit = CG == 2 ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / parts : blockIdx.x;
  const int units = CG == 2 ? gridDim.x >> 1 : SPLIT ? gridDim.x / parts : gridDim.x;
  const int all_kb = (p.K + kStep - 1) / kStep;
  const int first_kb = SPLIT ? all_kb * part / parts : 0;  // this CTA's steps (at least one: parts <= all_kb)
  const int num_kb = SPLIT ? all_kb * (part + 1) / parts - first_kb : all_kb;

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
  if (warp == 2) {
    const bool bad = load_offsets(p.offsets, p.groups, p.rows, off, status);
    if (lane == 0) bars->bad_offsets = bad;
    __syncwarp();
    if (!bad) scan_tiles<BT, MX4 ? Cfg::kBlockRows : 0>(off, p.groups, first, block);
  }
  tc_fence_before();
  if (CG == 2)
    gemm2::cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  volatile int* abort_flag = &bars->abort_flag;
  const RowsTable table{off, first, block};
  const int nt = (p.N + Cfg::kTileN - 1) / Cfg::kTileN;
  // bad offsets: no tile is computed (both CTAs of a pair read the same offsets)
  const int tiles = bars->bad_offsets ? 0 : first[p.groups] * nt;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      Ring<S> ring;
      uint32_t it = 0;
      bool ok = true;
      for (int i = unit; i < tiles && ok; i += units) {
        const RowsTile t = rows_locate<CG, BT, MX4>(p, table, i);
        const int a0 = t.n0 + int(rank) * 128;    // this CTA's weight rows
        const int share = t.mma_n / CG;
        const int b0 = t.r0 + int(rank) * share;  // and its share of the token rows
        const int boxes = (share + Cfg::kBox - 1) / Cfg::kBox;
        for (int kb = first_kb; kb < first_kb + num_kb; ++kb, ++it, ring.next()) {
          const int s = ring.s;
          if (!mbar_wait(&bars->empty[s], ring.phase ^ 1, status, 310)) { ok = false; *abort_flag = 1; break; }
          uint8_t* sa = smem + s * Cfg::kStageBytes;
          uint8_t* sb = sa + Cfg::kABytes;
          uint64_t* bar = &bars->full[s];
          if (rank == 0) mbar_arrive_expect_tx(bar, CG * (Cfg::kABytes + Cfg::kSfBytes + boxes * (Cfg::kBox * 128)));
          if (MX4) {
            uint8_t* sf = sb + Cfg::kBBytes;
            load_3d<CG>(sa, &p.tmA, bar, kb * 128, a0, t.g);
            for (int j = 0; j < boxes; ++j)
              load_2d<CG>(sb + j * (Cfg::kBox * 128), &p.tmB, bar, kb * 128, b0 + j * Cfg::kBox);
            const int ab = min(a0 >> 7, p.a_blocks - 1);  // a block past the matrix: any scales, the rows are not stored
            load_2d<CG>(sf, &p.tmSfa, bar, 0, (t.g * p.a_blocks + ab) * p.kpairs + kb);
#pragma unroll
            for (int j = 0; j < Cfg::kBlocksB; ++j)
              load_2d<CG>(sf + 1024 * (1 + j), &p.tmSfb, bar, 0, (t.block + (Cfg::kBlockRows * j < t.count ? j : 0)) * p.kpairs + kb);
          } else {
            const int k0 = kb * BK;
            if (!kAMn) {
              load_3d<CG>(sa, &p.tmA, bar, k0, a0, t.g);
            } else {
              load_3d<CG>(sa, &p.tmA, bar, a0, k0, t.g);
              load_3d<CG>(sa + BK * 128, &p.tmA, bar, a0 + 64, k0, t.g);
            }
            for (int j = 0; j < boxes; ++j)
              load_2d<CG>(sb + j * (Cfg::kBox * 128), &p.tmB, bar, k0, b0 + j * Cfg::kBox);
          }
        }
      }
      if (!ok && rank == 0) {
        // Drain: wait (bounded) for every stage that may still have bytes in flight.
        for (uint32_t j = (it >= S ? it - S : 0); j < it; ++j) mbar_wait(&bars->full[j % S], (j / S) & 1, status, 312);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && rank == 0) {
      Ring<S> ring;
      int tc = 0;
      bool ok = true, issued = false;
      const uint32_t smem0 = smem_u32(smem);
      const uint64_t a_desc = kAMn ? gemm::desc_mnmajor(smem0) : gemm::desc_kmajor(smem0);
      const uint64_t b_desc = gemm::desc_kmajor(smem0 + Cfg::kABytes);
      constexpr int kAStep = (kAMn ? 16 * 128 : 32) >> 4, kBStep = 32 >> 4;  // descriptor units per MMA
      for (int i = unit; i < tiles && ok; i += units) {
        const RowsTile t = rows_locate<CG, BT, MX4>(p, table, i);
        const int b = Cfg::kAccums == 2 ? (tc & 1) : 0;
        const int use = Cfg::kAccums == 2 ? (tc >> 1) : tc;
        if (!mbar_wait(&bars->tmem_empty[b], (use & 1) ^ 1, status, 320)) { ok = false; break; }
        tc_fence_after();
        const uint32_t dcol = tmem_base + b * BT;
        const uint32_t idesc = MX4 ? idesc_mxf4(128 * CG, t.mma_n)
                                   : (idesc_bf16(128 * CG, 0, kAMn, false) | (uint32_t(t.mma_n >> 3) << 17));
        for (int kb = 0; kb < num_kb; ++kb, ring.next()) {
          const int s = ring.s;
          if (!mbar_wait(&bars->full[s], ring.phase, status, 321)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = a_desc + uint32_t(s * (Cfg::kStageBytes >> 4));
          const uint64_t bd = b_desc + uint32_t(s * (Cfg::kStageBytes >> 4));
          if (MX4) {
            const uint32_t sf = smem0 + s * Cfg::kStageBytes + Cfg::kABytes + Cfg::kBBytes;
            const uint32_t sfa = tmem_base + Cfg::kAccums * BT + s * Cfg::kSfCols, sfb = sfa + 8;
            // columns: [atom 0 | atom 1] of A, then per atom the blocks of B side by side
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              copy_scales<CG>(sfa + 4 * c, sf + 512 * c);
#pragma unroll
              for (int j = 0; j < Cfg::kBlocksB; ++j)
                copy_scales<CG>(sfb + (c * Cfg::kBlocksB + j) * 4, sf + 1024 * (1 + j) + 512 * c);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_mxf4<CG>(dcol, ad + k * kAStep, bd + k * kBStep, idesc, sfa + 4 * (k >> 1),
                            sfb + 4 * Cfg::kBlocksB * (k >> 1), uint32_t(2 * (k & 1)), k != 0 || kb != 0 ? 1u : 0u);
          } else {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              issue<CG>(dcol, ad + k * kAStep, bd + k * kBStep, idesc, k != 0 || kb != 0 ? 1u : 0u);
          }
          issued = true;
          commit<CG>(&bars->empty[s]);
        }
        if (ok) commit<CG>(&bars->tmem_full[b]);
        ++tc;
      }
      if (!ok) *abort_flag = 1;
      // Every MMA has landed before TMEM is released.
      if (issued) {
        commit<CG>(&bars->drain);
        mbar_wait(&bars->drain, 0, status, 323);
      }
    }
  } else {
    // ---------------- Epilogue (warps 2..5) ----------------
    const int quarter = warp & 3;  // TMEM lanes [32*quarter, 32*quarter+32)
    RowsEpilogue<MODE> epi{p, smem_u32(epi_smem) + uint32_t(quarter * 2 * Cfg::kBuf)};
    if constexpr (SPLIT) {
      // fp32 of chunk c, this warp, fragment element j: 4 bytes per lane (the ring is free: its steps are summed)
      const uint32_t mine = smem_u32(smem) + uint32_t(quarter * 4096 + lane * 4);
      RowsTile t;
      bool ok = unit < tiles;
      if (ok) {
        t = rows_locate<CG, BT, MX4>(p, table, unit);
        ok = __all_sync(~0u, mbar_wait(&bars->tmem_full[0], 0, status, 330) && !*abort_flag);
        tc_fence_after();
      }
      const int col0 = ok ? t.n0 + quarter * 32 : p.N, chunks = ok ? (t.count + 31) / 32 : 0;
      const bool on = col0 < p.N;
      auto read = [&](int c, float (&v)[32]) {
        uint32_t lo[16], hi[16];
        const uint32_t acc = tmem_base + (uint32_t(quarter * 32) << 16) + c * 32;
        tmem_ld_16x256b_x4(acc, lo);
        tmem_ld_16x256b_x4(acc + (16u << 16), hi);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] = __uint_as_float(lo[j]);
          v[16 + j] = __uint_as_float(hi[j]);
        }
      };
      if (on) {
        for (int c = 0; c < chunks; ++c) {
          if (c % parts == part) continue;
          float v[32];
          read(c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + uint32_t(c * 16384 + j * 128)), "f"(v[j]) : "memory");
        }
      }
      cluster_barrier();
      if (on) {
        epi.tile_begin(t, col0);
        for (int c = part; c < chunks; c += parts) {
          uint4 aux[4];
          if (MODE == gemm::kGeluBwd) epi.load_aux(t.r0 + 32 * c, t.count - 32 * c, col0, aux);
          float v[32];
          read(c, v);
          for (int i = 0; i < parts; ++i) {
            if (i == part) continue;
            const uint32_t from = gemm2::mapa(mine + uint32_t(c * 16384), uint32_t(i));
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += load_cluster(from + uint32_t(j * 128));
          }
          epi.block(v, aux, t.r0 + 32 * c, t.count - 32 * c, col0);
        }
      }
      cluster_barrier();  // no CTA leaves while its sums are read
    }
    int tc = 0;
    for (int i = unit; !SPLIT && i < tiles; i += units) {
      const RowsTile t = rows_locate<CG, BT, MX4>(p, table, i);
      const int b = Cfg::kAccums == 2 ? (tc & 1) : 0;
      const int use = Cfg::kAccums == 2 ? (tc >> 1) : tc;
      const int col0 = t.n0 + int(rank) * 128 + quarter * 32;
      const bool on = col0 < p.N;
      uint4 aux[4];
      if (on) {
        epi.tile_begin(t, col0);
        if (MODE == gemm::kGeluBwd) epi.load_aux(t.r0, t.count, col0, aux);
      }
      bool ok = mbar_wait(&bars->tmem_full[b], use & 1, status, 330);
      if (*abort_flag) ok = false;
      if (!ok) { *abort_flag = 1; break; }
      tc_fence_after();
      const uint32_t acc = tmem_base + (uint32_t(quarter * 32) << 16) + b * BT;
      const int chunks = (t.count + 31) / 32;
      if constexpr (Cfg::kAccums == 1) {
        // The only accumulator: it is read whole (rounded to bf16, half the
        // registers) and given back to the MMAs before anything is stored.
        uint32_t w[BT / 32][16];
#pragma unroll
        for (int c = 0; c < BT / 32; ++c) {
          if (c < chunks && on) {
            uint32_t lo[16], hi[16];
            tmem_ld_16x256b_x4(acc + c * 32, lo);
            tmem_ld_16x256b_x4(acc + (16u << 16) + c * 32, hi);
            tmem_wait_ld();
            float v[32];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              v[j] = __uint_as_float(lo[j]);
              v[16 + j] = __uint_as_float(hi[j]);
            }
            epi.add_bias(v);
            epi.pack(v, w[c]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader<CG>(&bars->tmem_empty[b]);
#pragma unroll
        for (int c = 0; c < BT / 32; ++c) {
          if (c < chunks && on) {
            const uint32_t buf = epi.claim();
            epi.stage(buf, w[c]);
            epi.release(buf, t.r0 + 32 * c, t.count - 32 * c, col0);
          }
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          uint32_t lo[16], hi[16];
          if (on) {
            tmem_ld_16x256b_x4(acc + c * 32, lo);
            tmem_ld_16x256b_x4(acc + (16u << 16) + c * 32, hi);
            tmem_wait_ld();
          }
          if (c == chunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_leader<CG>(&bars->tmem_empty[b]);
          }
          if (!on) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            v[j] = __uint_as_float(lo[j]);
            v[16 + j] = __uint_as_float(hi[j]);
          }
          uint4 cur[4];
          if (MODE == gemm::kGeluBwd) {
#pragma unroll
            for (int j = 0; j < 4; ++j) cur[j] = aux[j];
            if (c + 1 < chunks) epi.load_aux(t.r0 + 32 * (c + 1), t.count - 32 * (c + 1), col0, aux);
          }
          epi.block(v, cur, t.r0 + 32 * c, t.count - 32 * c, col0);
        }
      }
      ++tc;
    }
    epi.finish();
  }

  if (SPLIT && warp < 2) {  // the epilogue's two barriers
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
