// Mixture-of-experts routing and row exchange.
//
// Router.  For a token with logits z[0..E) the k experts with the largest
// logits are chosen (ties: the lowest index) and weighted by
//   normalised:  w_j = exp(z_j - m) / sum_{i chosen} exp(z_i - m)
//   otherwise:   w_j = exp(z_j - m) / sum_{all e}    exp(z_e - m),   m = max z
// A row whose logits are all -inf gets weights 0 (not 0/0).  The gradient is
//   normalised:  dz_j = w_j (dw_j - sum_i w_i dw_i) on the chosen, 0 elsewhere
//   otherwise:   dz_e = p_e (dw_e [chosen] - sum_i w_i dw_i)
// The choices c = t*k + j are grouped by expert, stably: slots[c] is the row of
// choice c in the grouped order, order[slot] the choice of that row, and
// offsets[e] the first row of expert e.  Only integer atomics are used, so the
// result does not depend on the order of execution.
//
// Routing is bound by the instructions of the selection, not by memory: 16384
// tokens, 128 experts, top 8 take 16.3 us (two launches), 2^20 tokens 656 us
// (three), up to 128 tokens one launch of 4.5 us, the gradient 3.5 us.
//
// Exchange.  dispatch copies token rows to their k grouped rows, combine forms
// the weighted sum of a token's k rows; each is the other's gradient.  All four
// are bound by memory: one thread owns 8 columns of one token, so the token's
// row is read (or written) once whatever k is, and sums are in fp32 with one
// rounding to bf16 at the end.
#include "common.cuh"

namespace tdb {
namespace moe {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRouteThreads = 1024;    // routing: 32 warps
constexpr int kTokensPerBlock = 128;   // four tokens per warp; up to 128 tokens are routed by one launch
constexpr int kMaxTokens = 0x7fffffff - 1024;  // tokens of the block after the last one stay 32-bit
constexpr int kRankWarps = 8;          // warps that rank a block's choices

// Monotone map float -> uint32 (larger float, larger key); both zeros map to
// the same key, NaN to the largest.  Every key of a float is > 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = v == 0.f ? 0u : __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ float load_logit(const T* p);
template <>
__device__ __forceinline__ float load_logit<float>(const float* p) { return __ldg(p); }
template <>
__device__ __forceinline__ float load_logit<uint16_t>(const uint16_t* p) { return bf16_bits_to_float(__ldg(p)); }

// One warp: the top k of TT tokens at once (the rounds of one token depend on
// each other, those of several overlap).  Lane j < k returns the j-th choice's
// id and weight.  NP = experts per lane (expert i*32 + lane); rows past the
// last token repeat it.
template <int NP, int TT, typename T>
__device__ __forceinline__ void choose(const T* logits, int64_t ld, int t0, int t_step, int tokens, int E, int k,
                                       int normalize, int (&my_id)[TT], float (&my_w)[TT]) {
  const int lane = threadIdx.x & 31;
  float v[TT][NP];
  uint32_t key[TT][NP];
#pragma unroll
  for (int q = 0; q < TT; ++q) {
    const T* row = logits + int64_t(min(t0 + q * t_step, tokens - 1)) * ld;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int e = i * 32 + lane;
      v[q][i] = e < E ? load_logit<T>(row + e) : -INFINITY;
    }
  }
#pragma unroll
  for (int q = 0; q < TT; ++q)
#pragma unroll
    for (int i = 0; i < NP; ++i) key[q][i] = i * 32 + lane < E ? order_key(v[q][i]) : 0u;
  // Up to four experts per lane are sorted first (equal keys keep their order),
  // so a round looks at each lane's head only; more are searched every round.
  constexpr bool kSort = NP <= 4;
  int idx[TT][NP];
#pragma unroll
  for (int q = 0; q < TT; ++q) {
#pragma unroll
    for (int i = 0; i < NP; ++i) idx[q][i] = i * 32 + lane;
    if (kSort) {
#pragma unroll
      for (int end = NP - 1; end > 0; --end)
#pragma unroll
        for (int i = 0; i < end; ++i) {
          const bool swap = key[q][i + 1] > key[q][i];
          const uint32_t hi = swap ? key[q][i + 1] : key[q][i], lo = swap ? key[q][i] : key[q][i + 1];
          const int ih = swap ? idx[q][i + 1] : idx[q][i], il = swap ? idx[q][i] : idx[q][i + 1];
          key[q][i] = hi;
          key[q][i + 1] = lo;
          idx[q][i] = ih;
          idx[q][i + 1] = il;
        }
    }
  }
  uint32_t top_key[TT], my_key[TT];
  for (int j = 0; j < k; ++j) {
#pragma unroll
    for (int q = 0; q < TT; ++q) {
      uint32_t best = key[q][0];
      int at = idx[q][0];
      if (!kSort) {
#pragma unroll
        for (int i = 1; i < NP; ++i)
          if (key[q][i] > best) {
            best = key[q][i];
            at = idx[q][i];
          }
      }
      const uint32_t m = __reduce_max_sync(0xffffffffu, best);
      const uint32_t id = __reduce_min_sync(0xffffffffu, best == m ? uint32_t(at) : 0x7fffffffu);
      if ((id & 31u) == uint32_t(lane)) {
        if (kSort) {
#pragma unroll
          for (int i = 0; i + 1 < NP; ++i) {
            key[q][i] = key[q][i + 1];
            idx[q][i] = idx[q][i + 1];
          }
          key[q][NP - 1] = 0u;
        } else {
#pragma unroll
          for (int i = 0; i < NP; ++i)
            if (uint32_t(i) == id >> 5) key[q][i] = 0u;
        }
      }
      if (j == 0) top_key[q] = m;
      if (j == 0 || lane == j) {
        my_id[q] = int(id);
        my_key[q] = m;
      }
    }
  }
  float my_z[TT], top[TT];
#pragma unroll
  for (int q = 0; q < TT; ++q) {
    my_z[q] = key_value(my_key[q]);
    top[q] = key_value(top_key[q]);
  }
#pragma unroll
  for (int q = 0; q < TT; ++q) {
    const bool open = top[q] != -INFINITY;  // else no expert is open to this token
    const float e = open && lane < k ? expf(my_z[q] - top[q]) : 0.f;
    float part = e;
    if (!normalize) {
      part = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) part += i * 32 + lane < E ? expf(v[q][i] - top[q]) : 0.f;
    }
    const float s = warp_sum(part);
    my_w[q] = open ? e / s : 0.f;
  }
}

// Exclusive scan of total[0..E) into start[0..E], by one warp.
__device__ __forceinline__ void scan_experts(const int* total, int* start, int E) {
  const int lane = threadIdx.x & 31;
  const int per = (E + 31) / 32;
  int sum = 0;
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    if (e < E) sum += total[e];
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  int run = inc - sum;
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    if (e < E) {
      start[e] = run;
      run += total[e];
    }
  }
  if (lane == 31) start[E] = inc;
}

// Stable ranks of the block's `count` choices from c0 on: base[e] is the first
// slot of the block's choices of expert e.  Warp w < kRankWarps owns a contiguous
// share, so ranks follow the choice index.  wh: [kRankWarps][E] shared ints.
// ids: the block's choices in shared memory.  Indices count from c0, so that none
// leaves 32 bits where the last choices are near 2^31.
__device__ __forceinline__ void rank_choices(const int* ids, int c0, int count, int E, const int* base, int* wh,
                                             int* __restrict__ order, int* __restrict__ slots) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = ((count + kRankWarps - 1) / kRankWarps + 31) / 32 * 32;
  const int lo = warp < kRankWarps ? min(warp * share, count) : count, hi = min(lo + share, count);
  for (int i = threadIdx.x; i < kRankWarps * E; i += kRouteThreads) wh[i] = 0;
  __syncthreads();
  for (int c = lo + lane; c < hi; c += 32) atomicAdd(&wh[warp * E + ids[c]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    int run = base[e];
#pragma unroll
    for (int w = 0; w < kRankWarps; ++w) {
      const int n = wh[w * E + e];
      wh[w * E + e] = run;
      run += n;
    }
  }
  __syncthreads();
  for (int c = lo; c < hi; c += 32) {
    const int mine = c + lane;
    const bool on = mine < hi;
    const int id = on ? ids[mine] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    int first = 0;
    if (on) first = wh[warp * E + id];
    __syncwarp();
    if (on) {
      const int slot = first + __popc(same & ((1u << lane) - 1u));
      slots[c0 + mine] = slot;
      order[slot] = c0 + mine;
      if ((same >> lane) == 1u) wh[warp * E + id] = slot + 1;  // the last of its group
    }
    __syncwarp();
  }
}

// Top k, weights and the block's expert counts; with one block also the
// grouping (hist unused).
template <int NP, typename T>
__global__ void __launch_bounds__(kRouteThreads) choose_kernel(const T* __restrict__ logits, int64_t ld, int tokens, int E,
                                                               int k, int normalize, int* ids,
                                                               float* __restrict__ weights, int* __restrict__ hist,
                                                               int* __restrict__ offsets, int* __restrict__ order,
                                                               int* __restrict__ slots) {
  extern __shared__ int sh[];
  __shared__ int s_ids[kTokensPerBlock * kMaxTopK];
  int* count = sh;  // [E]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < E; e += kRouteThreads) count[e] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * kTokensPerBlock, t1 = min(t0 + kTokensPerBlock, tokens);
  constexpr int kStep = kRouteThreads / 32;
  constexpr int TT = NP <= 2 ? 4 : NP == 4 ? 2 : 1;  // 64 registers per thread
  for (int t = t0 + warp; t < t1; t += kStep * TT) {
    int id[TT];
    float w[TT];
    choose<NP, TT, T>(logits, ld, t, kStep, t1, E, k, normalize, id, w);
#pragma unroll
    for (int q = 0; q < TT; ++q) {
      const int tq = t + q * kStep;
      if (lane < k && tq < t1) {
        ids[int64_t(tq) * k + lane] = id[q];
        if (gridDim.x == 1) s_ids[tq * k + lane] = id[q];
        weights[int64_t(tq) * k + lane] = w[q];
        atomicAdd(&count[id[q]], 1);
      }
    }
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e < E; e += kRouteThreads) hist[int64_t(blockIdx.x) * E + e] = count[e];
    return;
  }
  int* start = sh + E;           // [E + 1]
  int* wh = start + E + 1;       // [kRankWarps][E]
  if (warp == 0) scan_experts(count, start, E);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kRouteThreads) offsets[e] = start[e];
  rank_choices(s_ids, 0, tokens * k, E, start, wh, order, slots);
}

// Running sums of the counts along the blocks, in place: hist[b][e] becomes the
// choices of expert e in the blocks up to b.  A block takes 8 experts (a row's
// 32 bytes) with 128 threads each; a thread reads its share of the rows twice,
// first for the shares' sums.
constexpr int kScanExperts = 8;
constexpr int kScanShares = kRouteThreads / kScanExperts;

__global__ void __launch_bounds__(kRouteThreads) scan_kernel(int* hist, int blocks, int E) {
  __shared__ int sums[kScanExperts][kScanShares];
  const int col = threadIdx.x % kScanExperts, share = threadIdx.x / kScanExperts;
  const int e = blockIdx.x * kScanExperts + col;
  const int per = (blocks + kScanShares - 1) / kScanShares;
  const int lo = min(share * per, blocks), hi = e < E ? min(lo + per, blocks) : lo;
  int* column = hist + e;
  int sum = 0;
#pragma unroll 8
  for (int b = lo; b < hi; ++b) sum += column[int64_t(b) * E];
  sums[col][share] = sum;
  __syncthreads();
  if (threadIdx.x < kScanExperts * 32) {  // a warp per expert, four shares per lane
    const int lane = threadIdx.x & 31;
    int* row = sums[threadIdx.x >> 5] + lane * 4;
    const int n[4] = {row[0], row[1], row[2], row[3]};
    const int all = n[0] + n[1] + n[2] + n[3];
    int run = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    run -= all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row[i] = run;
      run += n[i];
    }
  }
  __syncthreads();
  int run = sums[col][share];
  for (int b0 = lo; b0 < hi; b0 += 8) {
    int n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = b0 + i < hi ? column[int64_t(b0 + i) * E] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      run += n[i];
      if (b0 + i < hi) column[int64_t(b0 + i) * E] = run;
    }
  }
}

// Slots of one block's choices.  hist holds every block's counts, which each
// block adds up for itself, or (SCANNED) their running sums.
template <bool SCANNED>
__global__ void __launch_bounds__(kRouteThreads) group_kernel(const int* __restrict__ ids, const int* __restrict__ hist,
                                                              int blocks, int tokens, int E, int k,
                                                              int* __restrict__ offsets, int* __restrict__ order,
                                                              int* __restrict__ slots) {
  extern __shared__ int sh[];
  int* total = sh;          // [E]
  int* before = sh + E;     // [E]
  int* start = before + E;  // [E + 1]
  int* wh = start + E + 1;  // [kRankWarps][E]
  __shared__ int s_ids[kTokensPerBlock * kMaxTopK];
  const int t0 = blockIdx.x * kTokensPerBlock, t1 = min(t0 + kTokensPerBlock, tokens);
  for (int i = threadIdx.x; i < (t1 - t0) * k; i += kRouteThreads) s_ids[i] = ids[int64_t(t0) * k + i];
  if (SCANNED) {
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
      total[e] = __ldg(hist + int64_t(blocks - 1) * E + e);
      before[e] = blockIdx.x ? __ldg(hist + int64_t(blockIdx.x - 1) * E + e) : 0;
    }
  } else {
    for (int e = threadIdx.x; e < E; e += kRouteThreads) total[e] = before[e] = 0;
    __syncthreads();
    // A thread sums the counts of one expert over every `groups`-th block, eight
    // loads at a time (each is an L2 round trip).
    const int wide = (E + 31) / 32 * 32;
    const int groups = kRouteThreads / wide;
    const int part = threadIdx.x / wide, e = threadIdx.x % wide;
    if (part < groups && e < E) {
      int all = 0, mine = 0;
      for (int b0 = part; b0 < blocks; b0 += 8 * groups) {
        int n[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int b = b0 + i * groups;
          n[i] = b < blocks ? __ldg(hist + int64_t(b) * E + e) : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          all += n[i];
          mine += b0 + i * groups < int(blockIdx.x) ? n[i] : 0;
        }
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], mine);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) scan_experts(total, start, E);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= E; i += kRouteThreads) offsets[i] = start[i];
  for (int i = threadIdx.x; i < E; i += kRouteThreads) before[i] += start[i];
  __syncthreads();
  rank_choices(s_ids, t0 * k, (t1 - t0) * k, E, before, wh, order, slots);
}

__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = float_to_bf16_bits(v); }

// One warp per token.
template <int NP, typename T, typename O>
__global__ void __launch_bounds__(kThreads) route_bwd_kernel(const T* __restrict__ logits, int64_t ld, int tokens, int E,
                                                             int k, int normalize, const int* __restrict__ ids,
                                                             const float* __restrict__ weights,
                                                             const float* __restrict__ dweights, O* __restrict__ out,
                                                             int64_t ld_out) {
  const int lane = threadIdx.x & 31;
  const int64_t t = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= tokens) return;
  int id = -1;
  float w = 0.f, dw = 0.f;
  if (lane < k) {
    id = ids[t * k + lane];
    w = weights[t * k + lane];
    dw = dweights[t * k + lane];
  }
  const float dot = warp_sum(w * dw);
  O* o = out + t * ld_out;
  if (normalize) {
    // zeros, then the chosen ones over them (__syncwarp orders the two stores)
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (i * 32 + lane < E) store_logit(o + i * 32 + lane, 0.f);
    __syncwarp();
    if (uint32_t(id) < uint32_t(E)) store_logit(o + id, w * (dw - dot));
    return;
  }
  float z[NP], d[NP], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    z[i] = i * 32 + lane < E ? load_logit<T>(logits + t * ld + i * 32 + lane) : -INFINITY;
    top = fmaxf(top, z[i]);
    d[i] = -dot;
  }
#pragma unroll
  for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  for (int j = 0; j < k; ++j) {
    const int at = __shfl_sync(0xffffffffu, id, j);
    const float gj = __shfl_sync(0xffffffffu, dw, j);
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (at == i * 32 + lane) d[i] += gj;
  }
  float part = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    z[i] = top == -INFINITY ? 0.f : expf(z[i] - top);  // padding lanes: exp(-inf) = 0
    part += z[i];
  }
  const float s = warp_sum(part);
  const float inv = s > 0.f ? 1.f / s : (s == 0.f ? 0.f : s);  // all -inf: zero gradient; NaN stays NaN
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (i * 32 + lane < E) store_logit(o + i * 32 + lane, z[i] * inv * d[i]);
}

// ---------------------------------------------------------------------------
// Exchange.  Bound by the memory, so what matters is how many loads a thread
// has in flight: a block takes up to kTokens tokens per row of threads (a token
// narrower than the block takes only a part of its threads), reads all their
// slots at once, and each thread issues all its loads of a step before it uses
// any.  4096 tokens of 4096 columns, two choices each: dispatch 14.1 us (7.1 TB/s
// with L2's help), combine 15.0 us, its gradient 28.7 us (5.8 TB/s), the four
// directions of a training step together 82 us.
// ---------------------------------------------------------------------------
constexpr int kTokens = 4;  // at most; fewer where the tokens would not fill the SMs

__device__ __forceinline__ void unpack8(const uint4& q, float (&v)[8]) {
  const uint32_t a[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ uint4 load16(const uint16_t* row, int v) { return __ldg(reinterpret_cast<const uint4*>(row) + v); }

struct Choices {
  int slot[8 * kTokens][kMaxTopK];
  float w[8 * kTokens][kMaxTopK];
};

// The slots (and weights) of the block's tokens [t0, t0 + n) into shared
// memory; a slot outside the grouped rows is recorded and becomes -1.
__device__ __forceinline__ void load_choices(const int* __restrict__ slots, const float* __restrict__ weights, int64_t t0,
                                             int n, int tokens, int k, Choices& c, int* status) {
  const int threads = blockDim.x * blockDim.y;
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < n * k; i += threads) {
    const int tt = i / k, j = i - tt * k;
    int s = -1;
    float w = 0.f;
    if (t0 + tt < tokens) {
      s = slots[t0 * k + i];
      if (weights) w = weights[t0 * k + i];
      if (uint32_t(s) >= uint32_t(tokens) * uint32_t(k)) {
        record_status(status, kBadArgument, 200, int(t0 + tt), s);
        s = -1;
      }
    }
    c.slot[tt][j] = s;
    c.w[tt][j] = w;
  }
  __syncthreads();
}

// U: 16-byte pieces of a row per thread and step.
constexpr int kDispatchPieces = 4;

__global__ void __launch_bounds__(kThreads) dispatch_kernel(const uint16_t* __restrict__ x, int64_t ldx, int tokens, int k,
                                                            int vecs, int turns, const int* __restrict__ slots,
                                                            uint16_t* __restrict__ out, int64_t ldo, int* status) {
  constexpr int U = kDispatchPieces;
  __shared__ Choices c;
  const int per = blockDim.y * turns;
  const int64_t t0 = int64_t(blockIdx.x) * per;
  load_choices(slots, nullptr, t0, per, tokens, k, c, status);
  for (int tt = threadIdx.y; tt < per && t0 + tt < tokens; tt += blockDim.y) {
    const uint16_t* src = x + (t0 + tt) * ldx;
    for (int v = threadIdx.x; v < vecs; v += U * blockDim.x) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = v + u * blockDim.x;
        if (at < vecs) q[u] = load16(src, at);
      }
      for (int j = 0; j < k; ++j) {
        const int s = c.slot[tt][j];
        if (s < 0) continue;
        uint4* dst = reinterpret_cast<uint4*>(out + int64_t(s) * ldo);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = v + u * blockDim.x;
          if (at < vecs) dst[at] = q[u];
        }
      }
    }
  }
}

// Pieces per thread when KC >= k rows are read for each: eight loads in flight.
template <int KC>
constexpr int kCombinePieces = KC >= 8 ? 1 : 8 / KC;

// out[t] = residual[t] + sum_j w_j y[slot_j] (weights null: all 1).
template <int KC>
__global__ void __launch_bounds__(kThreads) combine_kernel(const uint16_t* __restrict__ y, int64_t ldy, int tokens, int k,
                                                           int vecs, int turns, const int* __restrict__ slots,
                                                           const float* __restrict__ weights,
                                                           const uint16_t* __restrict__ residual, int64_t ldr,
                                                           uint16_t* __restrict__ out, int64_t ldo, int* status) {
  constexpr int U = kCombinePieces<KC>;
  __shared__ Choices c;
  const int per = blockDim.y * turns;
  const int64_t t0 = int64_t(blockIdx.x) * per;
  load_choices(slots, weights, t0, per, tokens, k, c, status);
  for (int tt = threadIdx.y; tt < per && t0 + tt < tokens; tt += blockDim.y) {
    for (int v = threadIdx.x; v < vecs; v += U * blockDim.x) {
      uint4 q[U][KC];
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const int s = j < k ? c.slot[tt][j] : -1;
        const uint16_t* row = y + int64_t(s) * ldy;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = v + u * blockDim.x;
          q[u][j] = make_uint4(0, 0, 0, 0);
          if (s >= 0 && at < vecs) q[u][j] = load16(row, at);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = v + u * blockDim.x;
        if (at >= vecs) break;
        float acc[8] = {}, f[8];
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          if (j >= k) break;
          const float w = weights ? c.w[tt][j] : 1.f;
          unpack8(q[u][j], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += w * f[e];
        }
        if (residual) {
          unpack8(load16(residual + (t0 + tt) * ldr, at), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += f[e];
        }
        reinterpret_cast<uint4*>(out + (t0 + tt) * ldo)[at] = pack8(acc);
      }
    }
  }
}

// dy[slot_j] = w_j dout[t];  dw_j = <dout[t], y[slot_j]> (fp32).
template <int KC>
__global__ void __launch_bounds__(kThreads) combine_bwd_kernel(const uint16_t* __restrict__ dout, int64_t ldd,
                                                               const uint16_t* __restrict__ y, int64_t ldy, int tokens,
                                                               int k, int vecs, int turns, const int* __restrict__ slots,
                                                               const float* __restrict__ weights,
                                                               uint16_t* __restrict__ dy, int64_t lddy,
                                                               float* __restrict__ dweights, int* status) {
  constexpr int U = kCombinePieces<KC>;
  __shared__ Choices c;
  __shared__ float s_dot[kTokens][kWarps][kMaxTopK];
  const int per = blockDim.y * turns;
  const int64_t t0 = int64_t(blockIdx.x) * per;
  load_choices(slots, weights, t0, per, tokens, k, c, status);
  const int lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5, warp = threadIdx.y * warps + (threadIdx.x >> 5);
#pragma unroll 1
  for (int r = 0; r < turns; ++r) {
    const int tt = r * blockDim.y + threadIdx.y;
    float dot[KC] = {};
    if (t0 + tt < tokens) {
      const uint16_t* src = dout + (t0 + tt) * ldd;
      for (int v = threadIdx.x; v < vecs; v += U * blockDim.x) {
        uint4 q[U][KC], qd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = v + u * blockDim.x;
          qd[u] = make_uint4(0, 0, 0, 0);
          if (at < vecs) qd[u] = load16(src, at);
        }
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          const int s = j < k ? c.slot[tt][j] : -1;
          const uint16_t* row = y + int64_t(s) * ldy;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int at = v + u * blockDim.x;
            q[u][j] = make_uint4(0, 0, 0, 0);
            if (s >= 0 && at < vecs) q[u][j] = load16(row, at);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = v + u * blockDim.x;
          if (at >= vecs) break;
          float d[8], f[8];
          unpack8(qd[u], d);
#pragma unroll
          for (int j = 0; j < KC; ++j) {
            if (j >= k) break;
            const int s = c.slot[tt][j];
            if (s < 0) continue;
            const float w = c.w[tt][j];
            unpack8(q[u][j], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              dot[j] += d[e] * f[e];
              f[e] = w * d[e];
            }
            reinterpret_cast<uint4*>(dy + int64_t(s) * lddy)[at] = pack8(f);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      if (j >= k) break;
      const float sum = warp_sum(dot[j]);
      if (lane == 0) s_dot[r][warp][j] = sum;
    }
  }
  __syncthreads();
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < per * k; i += blockDim.x * blockDim.y) {
    const int tt = i / k, j = i - tt * k;
    if (t0 + tt >= tokens) break;
    float sum = 0.f;
    for (int w = 0; w < warps; ++w) sum += s_dot[tt / blockDim.y][(tt % blockDim.y) * warps + w][j];
    dweights[t0 * k + i] = sum;
  }
}

// Threads of a token, each with `pieces` pieces of its row, and tokens of a block.
static dim3 exchange_block(int vecs, int pieces) {
  int x = ((vecs + pieces - 1) / pieces + 31) / 32 * 32;
  if (x > kThreads) x = kThreads;
  int y = kThreads / x;
  return dim3(x, y > 8 ? 8 : y);
}

// Tokens per row of threads: more than one only while the blocks still fill
// every SM eight times (2048 threads).
static int exchange_turns(int tokens, const dim3& block) {
  const int64_t turns = tokens / (int64_t(block.y) * tdb_host::sm_count() * 8);
  return turns < 1 ? 1 : turns > kTokens ? kTokens : int(turns);
}
static unsigned exchange_grid(int tokens, const dim3& block, int turns) {
  const int per = int(block.y) * turns;
  return unsigned((int64_t(tokens) + per - 1) / per);
}

static bool bad_rows(const void* p, int64_t ld, int H) {
  return !p || reinterpret_cast<uintptr_t>(p) % 16 || ld % 8 || ld < H;
}

// Whether the blocks' counts are summed once, by a launch of its own, instead of
// by every block of group_kernel, whose reads grow with the square of the
// tokens.  Microseconds of the whole call, by every block / once: 128 experts,
// top 8, 16384 tokens 16.4 / 16.9, 24576 28.0 / 26.5, 65536 65 / 49, 2^20 4697 /
// 656; 8 experts, top 2, 32768 15.8 / 16.2, 65536 31 / 28; 512 experts, top 8,
// 4096 38.8 / 39.3, 16384 42.6 / 39.9.
static bool scan_counts(int blocks, int E) { return blocks > 256 || int64_t(blocks) * E > 16384; }

template <typename T>
static int route(const T* logits, int64_t ld, int tokens, int E, int k, int normalize, int* ids, float* weights,
                 int* offsets, int* order, int* slots, int* hist, cudaStream_t s) {
  const int blocks = tokens > 0 ? (tokens + kTokensPerBlock - 1) / kTokensPerBlock : 1;
  const size_t one = size_t(2 * E + 1 + kRankWarps * E) * 4, many = size_t(E) * 4;
  const size_t smem = blocks == 1 ? one : many;
#define TDB_CHOOSE(NP) \
  choose_kernel<NP, T><<<blocks, kRouteThreads, smem, s>>>(logits, ld, tokens, E, k, normalize, ids, weights, hist, offsets, order, slots)
  if (E <= 32) TDB_CHOOSE(1);
  else if (E <= 64) TDB_CHOOSE(2);
  else if (E <= 128) TDB_CHOOSE(4);
  else if (E <= 256) TDB_CHOOSE(8);
  else TDB_CHOOSE(16);
#undef TDB_CHOOSE
  tdb_host::launched(1);
  if (blocks > 1) {
    const size_t tables = size_t(3 * E + 1 + kRankWarps * E) * 4;
    if (scan_counts(blocks, E)) {
      scan_kernel<<<(E + kScanExperts - 1) / kScanExperts, kRouteThreads, 0, s>>>(hist, blocks, E);
      group_kernel<true><<<blocks, kRouteThreads, tables, s>>>(ids, hist, blocks, tokens, E, k, offsets, order, slots);
      tdb_host::launched(2);
    } else {
      group_kernel<false><<<blocks, kRouteThreads, tables, s>>>(ids, hist, blocks, tokens, E, k, offsets, order, slots);
      tdb_host::launched(1);
    }
  }
  return int(cudaGetLastError());
}

template <typename T, typename O>
static int route_bwd(const T* logits, int64_t ld, int tokens, int E, int k, int normalize, const int* ids,
                     const float* weights, const float* dweights, O* out, int64_t ld_out, cudaStream_t s) {
  const int blocks = (tokens + kWarps - 1) / kWarps;
#define TDB_BWD(NP) \
  route_bwd_kernel<NP, T, O><<<blocks, kThreads, 0, s>>>(logits, ld, tokens, E, k, normalize, ids, weights, dweights, out, ld_out)
  if (E <= 32) TDB_BWD(1);
  else if (E <= 64) TDB_BWD(2);
  else if (E <= 128) TDB_BWD(4);
  else if (E <= 256) TDB_BWD(8);
  else TDB_BWD(16);
#undef TDB_BWD
  tdb_host::launched(1);
  return int(cudaGetLastError());
}

static int check_route(const char* what, int64_t ld, int tokens, int E, int k) {
  if (tokens < 0 || E < 1 || E > kMaxExperts || k < 1 || k > kMaxTopK || k > E || ld < E ||
      int64_t(tokens) * k >= (int64_t(1) << 31) || tokens > kMaxTokens)
    return tdb_host::fail(int(cudaErrorInvalidValue),
                          "%s: 1..%d experts, 1..%d choices per token (at most the experts), tokens * choices < 2^31, at "
                          "most %d tokens", what, kMaxExperts, kMaxTopK, kMaxTokens);
  return 0;
}

static int check_exchange(const char* what, int tokens, int k, int H) {
  if (tokens < 0 || k < 1 || k > kMaxTopK || H < 8 || H % 8 || int64_t(tokens) * k >= (int64_t(1) << 31))
    return tdb_host::fail(int(cudaErrorInvalidValue), "%s: 1..%d choices per token, columns a multiple of 8", what,
                          kMaxTopK);
  return 0;
}

static int bad_alignment(const char* what) {
  return tdb_host::fail(int(cudaErrorInvalidValue), "%s: rows must be 16-byte aligned and at least as wide as the columns", what);
}

}  // namespace moe
}  // namespace tdb

using namespace tdb;
using namespace tdb::moe;

// Ints of scratch that tdb_moe_route needs (0: none).
TDB_API long long tdb_moe_route_scratch_ints(int tokens, int E) {
  const int64_t blocks = (int64_t(tokens) + kTokensPerBlock - 1) / kTokensPerBlock;
  return blocks > 1 ? blocks * E : 0;
}

// logits fp32 (logits_bf16 = 0) or bf16 [tokens, E] (row stride ld) -> ids,
// weights, slots, order [tokens * k], offsets [E + 1].
TDB_API int tdb_moe_route(const void* logits, int logits_bf16, int64_t ld, int tokens, int E, int k, int normalize,
                          int* ids, float* weights, int* offsets, int* order, int* slots, int* scratch, void* stream) {
  if (int rc = check_route("moe route", ld, tokens, E, k)) return rc;
  if (!offsets || (tokens > 0 && (!logits || !ids || !weights || !order || !slots)) ||
      (tokens > kTokensPerBlock && !scratch))
    return tdb_host::fail(int(cudaErrorInvalidValue), "moe route: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_bf16)
    return route(static_cast<const uint16_t*>(logits), ld, tokens, E, k, normalize, ids, weights, offsets, order, slots,
                 scratch, s);
  return route(static_cast<const float*>(logits), ld, tokens, E, k, normalize, ids, weights, offsets, order, slots,
               scratch, s);
}

// dlogits (fp32 or bf16, [tokens, E], row stride ld_out) from dweights; the
// logits are read only when the weights were not normalised.
TDB_API int tdb_moe_route_bwd(const void* logits, int logits_bf16, int64_t ld, int tokens, int E, int k, int normalize,
                              const int* ids, const float* weights, const float* dweights, void* dlogits, int out_bf16,
                              int64_t ld_out, void* stream) {
  if (int rc = check_route("moe route backward", ld < ld_out ? ld : ld_out, tokens, E, k)) return rc;
  if (tokens == 0) return 0;
  if (!logits || !ids || !weights || !dweights || !dlogits)
    return tdb_host::fail(int(cudaErrorInvalidValue), "moe route backward: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_bf16) {
    const uint16_t* z = static_cast<const uint16_t*>(logits);
    return out_bf16 ? route_bwd(z, ld, tokens, E, k, normalize, ids, weights, dweights, static_cast<uint16_t*>(dlogits), ld_out, s)
                    : route_bwd(z, ld, tokens, E, k, normalize, ids, weights, dweights, static_cast<float*>(dlogits), ld_out, s);
  }
  const float* z = static_cast<const float*>(logits);
  return out_bf16 ? route_bwd(z, ld, tokens, E, k, normalize, ids, weights, dweights, static_cast<uint16_t*>(dlogits), ld_out, s)
                  : route_bwd(z, ld, tokens, E, k, normalize, ids, weights, dweights, static_cast<float*>(dlogits), ld_out, s);
}

// out[slots[t*k + j]] = x[t] (bf16 rows of H columns).
TDB_API int tdb_moe_dispatch(const void* x, int64_t ldx, int tokens, int k, int H, const int* slots, void* out,
                             int64_t ldo, void* stream) {
  if (int rc = check_exchange("moe dispatch", tokens, k, H)) return rc;
  if (tokens == 0) return 0;
  if (!slots || bad_rows(x, ldx, H) || bad_rows(out, ldo, H)) return bad_alignment("moe dispatch");
  const dim3 block = exchange_block(H / 8, kDispatchPieces);
  const int turns = exchange_turns(tokens, block);
  dispatch_kernel<<<exchange_grid(tokens, block, turns), block, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint16_t*>(x), ldx, tokens, k, H / 8, turns, slots, static_cast<uint16_t*>(out), ldo,
      tdb_host::status_ptr());
  tdb_host::launched(1);
  return int(cudaGetLastError());
}

// out[t] = (residual[t]) + sum_j (weights[t*k + j] or 1) * y[slots[t*k + j]].
TDB_API int tdb_moe_combine(const void* y, int64_t ldy, int tokens, int k, int H, const int* slots, const float* weights,
                            const void* residual, int64_t ldr, void* out, int64_t ldo, void* stream) {
  if (int rc = check_exchange("moe combine", tokens, k, H)) return rc;
  if (tokens == 0) return 0;
  if (!slots || bad_rows(y, ldy, H) || bad_rows(out, ldo, H) || (residual && bad_rows(residual, ldr, H)))
    return bad_alignment("moe combine");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define TDB_COMBINE(KC)                                                                                              \
  {                                                                                                                  \
    const dim3 block = exchange_block(H / 8, kCombinePieces<KC>);                                                    \
    const int turns = exchange_turns(tokens, block);                                                                 \
    combine_kernel<KC><<<exchange_grid(tokens, block, turns), block, 0, s>>>(                                        \
        static_cast<const uint16_t*>(y), ldy, tokens, k, H / 8, turns, slots, weights,                               \
        static_cast<const uint16_t*>(residual), ldr, static_cast<uint16_t*>(out), ldo, tdb_host::status_ptr());      \
  }
  if (k == 1) TDB_COMBINE(1)
  else if (k == 2) TDB_COMBINE(2)
  else if (k <= 4) TDB_COMBINE(4)
  else if (k <= 8) TDB_COMBINE(8)
  else TDB_COMBINE(16)
#undef TDB_COMBINE
  tdb_host::launched(1);
  return int(cudaGetLastError());
}

// Gradients of tdb_moe_combine: dy (grouped rows) and dweights [tokens * k].
TDB_API int tdb_moe_combine_bwd(const void* dout, int64_t ldd, const void* y, int64_t ldy, int tokens, int k, int H,
                                const int* slots, const float* weights, void* dy, int64_t lddy, float* dweights,
                                void* stream) {
  if (int rc = check_exchange("moe combine backward", tokens, k, H)) return rc;
  if (tokens == 0) return 0;
  if (!slots || !weights || !dweights || bad_rows(dout, ldd, H) || bad_rows(y, ldy, H) || bad_rows(dy, lddy, H))
    return bad_alignment("moe combine backward");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define TDB_COMBINE_BWD(KC)                                                                                          \
  {                                                                                                                  \
    const dim3 block = exchange_block(H / 8, kCombinePieces<KC>);                                                    \
    const int turns = exchange_turns(tokens, block);                                                                 \
    combine_bwd_kernel<KC><<<exchange_grid(tokens, block, turns), block, 0, s>>>(                                    \
        static_cast<const uint16_t*>(dout), ldd, static_cast<const uint16_t*>(y), ldy, tokens, k, H / 8, turns,      \
        slots, weights, static_cast<uint16_t*>(dy), lddy, dweights, tdb_host::status_ptr());                         \
  }
  if (k == 1) TDB_COMBINE_BWD(1)
  else if (k == 2) TDB_COMBINE_BWD(2)
  else if (k <= 4) TDB_COMBINE_BWD(4)
  else if (k <= 8) TDB_COMBINE_BWD(8)
  else TDB_COMBINE_BWD(16)
#undef TDB_COMBINE_BWD
  tdb_host::launched(1);
  return int(cudaGetLastError());
}
