// Grouped forward product for few rows (generated tokens): Y[r, n] = sum_k
// W_g[n, k] X[r, k] with at most kFewRows rows in all.
//
// Bound by reading each used W_g once, so the weights stream from global memory
// straight into the fragments of mma.sync m16n8k16 (the multiplications are
// few; tcgen05 would need them in shared memory first).  A sum over k may take
// the k in any order: a lane loads 8 consecutive k of a row in one 16-byte
// load and uses them as the k slots that the fragment layout gives it in two
// MMAs, for the weights (16 output columns as M) and the rows (8 as N) alike.
//
// A unit is 16 output columns of one group; the 8 warps of a block split K in
// turns of 32 (together 512 contiguous bytes of each weight row) and their sums
// are added in a fixed order.  Blocks stay and take unit after unit.  Every lane
// copies the pieces that it will use itself into its own slots of a ring in
// shared memory (cp.async, up to 12 turns ahead, across units), so two blocks
// keep some 190 KB of an SM's loads in flight and wait for no other thread.
// One token through two experts of 4096 x 4096: 17.3 us (3.9 TB/s), through one of
// 1024 x 1024 3.6 us (the tcgen05 tiles, sums shared: 18.2 and 8.2 us); of larger
// weights the tiles read faster (see pick_tile in grouped.cu).
#pragma once
#include "grouped_rows.cuh"

namespace tdb {
namespace grouped {

constexpr int kFewRows = 16;
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewTurns = 4;   // turns per step: one copy group, one round of the loop
constexpr int kFewDepth = 3;   // steps in the ring
constexpr int kFewRing = kFewDepth * kFewTurns * kFewThreads * 32;  // bytes

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes global -> shared, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t* src, bool on) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ uint4 read16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src));
  return v;
}

template <int MODE>
__global__ void __launch_bounds__(kFewThreads, 2) few_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx,
                                                                  const uint16_t* __restrict__ w,
                                                                  const int* __restrict__ offsets, int groups, int rows,
                                                                  int N, int K, const uint16_t* __restrict__ bias,
                                                                  uint16_t* __restrict__ out, int64_t ldo,
                                                                  uint16_t* __restrict__ pre, int64_t ldp, int* status) {
  extern __shared__ __align__(16) uint8_t ring_raw[];
  __shared__ int s_group[kFewRows], s_lo[kFewRows], s_hi[kFewRows], s_used;
  __shared__ float part[kFewWarps][kFewRows][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    // the groups with rows (at most kFewRows), and the check of all offsets
    bool bad = false;
    int used = 0, last = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
      const int g = g0 + lane;
      const int a = g < groups ? __ldg(offsets + g) : rows, b = g < groups ? __ldg(offsets + g + 1) : rows;
      bad |= a < last || b < a || b > rows;
      const bool has = g < groups && b > a;
      const uint32_t some = __ballot_sync(0xffffffffu, has);
      const int at = used + __popc(some & ((1u << lane) - 1u));
      if (has && at < kFewRows) {
        s_group[at] = g;
        s_lo[at] = a;
        s_hi[at] = b;
      }
      used += __popc(some);
      last = __shfl_sync(0xffffffffu, b, 31);
    }
    if (bad) record_status(status, kBadArgument, 300, groups, rows);
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) s_used = bad ? 0 : used;
  }
  __syncthreads();
  const int blocks_n = (N + 15) / 16;
  const int units = s_used * blocks_n;
  constexpr int kTurn = kFewWarps * 32;  // k per turn of the block
  constexpr int kStep = kFewTurns * kTurn;
  const int row = lane >> 2, col = (lane & 3) * 8 + warp * 32;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint32_t slot0 = smem_u32(ring_raw) + threadIdx.x * 16;
  constexpr uint32_t kHalf = kFewThreads * 16, kSlot = 2 * kHalf, kGroup = kFewTurns * kSlot;

  // what is copied next: the step at c_k of unit c_unit into ring position c_slot
  int c_unit = blockIdx.x, c_k = col;
  uint32_t c_slot = slot0;
  const uint16_t *c_a = w, *c_b = w;
  bool on_a = false, on_b = false;
  auto aim = [&]() {
    if (c_unit >= units) {
      on_a = on_b = false;
      c_a = c_b = w;
      return;
    }
    const int n = c_unit % blocks_n * 16 + row;
    on_a = n < N;
    on_b = n + 8 < N;
    c_a = on_a ? w + (int64_t(s_group[c_unit / blocks_n]) * N + n) * K : w;
    c_b = on_b ? c_a + int64_t(8) * K : w;
  };
  auto copy = [&]() {
    if (c_unit < units) {
#pragma unroll
      for (int u = 0; u < kFewTurns; ++u) {
        const int k = c_k + u * kTurn;
        const bool in = k < K;
        copy16(c_slot + u * kSlot, c_a + (in ? k : 0), in && on_a);
        copy16(c_slot + u * kSlot + kHalf, c_b + (in ? k : 0), in && on_b);
      }
      c_k += kStep;
      if (c_k - col >= K) {
        c_k = col;
        c_unit += gridDim.x;
        aim();
      }
    }
    c_slot = c_slot + kGroup == slot0 + kFewDepth * kGroup ? slot0 : c_slot + kGroup;
    asm volatile("cp.async.commit_group;" ::: "memory");  // one group per step, also where it is empty
  };
  aim();
#pragma unroll 1
  for (int i = 0; i < kFewDepth - 1; ++i) copy();

  uint32_t slot = slot0;
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int which = unit / blocks_n;
    const int r0 = s_lo[which], count = s_hi[which] - r0;  // 1..kFewRows
    const uint16_t* xa = x + int64_t(r0 + row) * ldx;
    float acc[2][4] = {};
    for (int k0 = col; k0 - col < K; k0 += kStep) {
      uint4 p[kFewTurns];
#pragma unroll
      for (int u = 0; u < kFewTurns; ++u)
        p[u] = row < count && k0 + u * kTurn < K ? __ldg(reinterpret_cast<const uint4*>(xa + k0 + u * kTurn)) : zero;
      asm volatile("cp.async.wait_group %0;" ::"n"(kFewDepth - 2) : "memory");
      uint4 a[kFewTurns], b[kFewTurns];
#pragma unroll
      for (int u = 0; u < kFewTurns; ++u) {
        a[u] = read16(slot + u * kSlot);
        b[u] = read16(slot + u * kSlot + kHalf);
      }
      slot = slot + kGroup == slot0 + kFewDepth * kGroup ? slot0 : slot + kGroup;
      copy();
#pragma unroll
      for (int u = 0; u < kFewTurns; ++u) {
        mma_bf16(acc[0], a[u].x, b[u].x, a[u].y, b[u].y, p[u].x, p[u].y);
        mma_bf16(acc[0], a[u].z, b[u].z, a[u].w, b[u].w, p[u].z, p[u].w);
      }
      if (count > 8) {
#pragma unroll
        for (int u = 0; u < kFewTurns; ++u)
          p[u] = row + 8 < count && k0 + u * kTurn < K
                     ? __ldg(reinterpret_cast<const uint4*>(xa + 8 * ldx + k0 + u * kTurn))
                     : zero;
#pragma unroll
        for (int u = 0; u < kFewTurns; ++u) {
          mma_bf16(acc[1], a[u].x, b[u].x, a[u].y, b[u].y, p[u].x, p[u].y);
          mma_bf16(acc[1], a[u].z, b[u].z, a[u].w, b[u].w, p[u].z, p[u].w);
        }
      }
    }
    // accumulator: columns row (+ 8) of the unit, rows 2 (lane % 4) + {0, 1} (+ 8)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[warp][8 * h + 2 * (lane & 3) + (e & 1)][row + 8 * (e >> 1)] = acc[h][e];
    __syncthreads();
    const int r = threadIdx.x >> 4, n = unit % blocks_n * 16 + (threadIdx.x & 15);
    if (r < count && n < N) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kFewWarps; ++i) v += part[i][r][threadIdx.x & 15];
      if (bias) v += bf16_bits_to_float(__ldg(bias + int64_t(s_group[which]) * N + n));
      if (MODE == gemm::kBiasGelu) {
        pre[int64_t(r0 + r) * ldp + n] = float_to_bf16_bits(v);
        v = gelu(v);
      }
      out[int64_t(r0 + r) * ldo + n] = float_to_bf16_bits(v);
    }
    __syncthreads();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace grouped
}  // namespace tdb
