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
// are added in a fixed order.  Blocks stay and take unit after unit, so that
// weights are always on their way.
#pragma once
#include "grouped_rows.cuh"

namespace tdb {
namespace grouped {

constexpr int kFewRows = 16;
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewTurns = 4;  // turns of 32 k whose loads are issued together

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_stream(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The weights of one step of a lane: kFewTurns turns of two rows.
struct FewWeights {
  uint4 a[kFewTurns], b[kFewTurns];
};

template <int MODE>
__global__ void __launch_bounds__(kFewThreads, 2) few_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx,
                                                                  const uint16_t* __restrict__ w,
                                                                  const int* __restrict__ offsets, int groups, int rows,
                                                                  int N, int K, const uint16_t* __restrict__ bias,
                                                                  uint16_t* __restrict__ out, int64_t ldo,
                                                                  uint16_t* __restrict__ pre, int64_t ldp, int* status) {
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
  constexpr int kStep = kFewTurns * kFewWarps * 32;  // k per step of the block
  const int steps = (K + kStep - 1) / kStep;
  const int row = lane >> 2, col = (lane & 3) * 8 + warp * 32;
  const uint4 zero = make_uint4(0, 0, 0, 0);

  auto load = [&](int unit, int step, FewWeights& f) {
    if (unit >= units) return;
    const int n = unit % blocks_n * 16 + row;
    const uint16_t* wa = w + (int64_t(s_group[unit / blocks_n]) * N + n) * K + col + step * kStep;
#pragma unroll
    for (int u = 0; u < kFewTurns; ++u) {
      const bool in = step * kStep + u * kFewWarps * 32 + col < K;
      f.a[u] = in && n < N ? load_stream(wa + u * kFewWarps * 32) : zero;
      f.b[u] = in && n + 8 < N ? load_stream(wa + int64_t(8) * K + u * kFewWarps * 32) : zero;
    }
  };

  FewWeights next;
  load(blockIdx.x, 0, next);
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int slot = unit / blocks_n;
    const int r0 = s_lo[slot], count = s_hi[slot] - r0;  // 1..kFewRows
    const uint16_t* xa = x + int64_t(r0 + row) * ldx + col;
    float acc[2][4] = {};
    for (int step = 0; step < steps; ++step) {
      const FewWeights f = next;
      // the next step's weights, this unit's or the next one's, are on their way during the MMAs and the sums
      if (step + 1 < steps)
        load(unit, step + 1, next);
      else
        load(unit + gridDim.x, 0, next);
#pragma unroll
      for (int u = 0; u < kFewTurns; ++u) {
        const int k = step * kStep + u * kFewWarps * 32;
        const bool in = k + col < K;
        const uint4 p = in && row < count ? __ldg(reinterpret_cast<const uint4*>(xa + k)) : zero;
        mma_bf16(acc[0], f.a[u].x, f.b[u].x, f.a[u].y, f.b[u].y, p.x, p.y);
        mma_bf16(acc[0], f.a[u].z, f.b[u].z, f.a[u].w, f.b[u].w, p.z, p.w);
        if (count > 8) {
          const uint4 q = in && row + 8 < count ? __ldg(reinterpret_cast<const uint4*>(xa + 8 * ldx + k)) : zero;
          mma_bf16(acc[1], f.a[u].x, f.b[u].x, f.a[u].y, f.b[u].y, q.x, q.y);
          mma_bf16(acc[1], f.a[u].z, f.b[u].z, f.a[u].w, f.b[u].w, q.z, q.w);
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
      if (bias) v += bf16_bits_to_float(__ldg(bias + int64_t(s_group[slot]) * N + n));
      if (MODE == gemm::kBiasGelu) {
        pre[int64_t(r0 + r) * ldp + n] = float_to_bf16_bits(v);
        v = gelu(v);
      }
      out[int64_t(r0 + r) * ldo + n] = float_to_bf16_bits(v);
    }
    __syncthreads();
  }
}

}  // namespace grouped
}  // namespace tdb
