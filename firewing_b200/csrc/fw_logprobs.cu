// fw_logprobs.cu -- log probabilities of given tokens, entropy and the top
// alternatives of rows of logits (fw_token_logprobs).
//
// For a row z[0..V), c = log2(e) / temperature and a reference M near the
// row's maximum, with y_i = (z_i - M) c:
//   S = sum 2^y_i,  W = sum 2^y_i y_i
//   log p_i = (z_i - M) / temperature - ln S,  H = ln 2 (log2 S - W / S)
// S and W are sums of f32 terms that any part of the row adds up against a
// reference of its own; parts are joined by rescaling, and carry S - 1, without
// the maximum's own term: a row that is sure of one token has a log S far
// below the rounding of S.  One pass over the
// row keeps S, W and the candidates for the alternatives.
//
// The reference is the warp's maximum so far: with one far below the row's,
// log2 S and W / S would be large and nearly equal, and their difference, the
// entropy, inexact.  It changes about log(batches) times per row, one vote per
// batch.
// The alternatives: K values at least are >= `floor` (publish_share), taken from
// the first batch and raised after 1, 2, 4, ... of them.  Values under it cost
// one comparison per lane and batch; the few others go to a list in shared
// memory.  A list that overflows (a row of equal values, an ascending row) is
// made anew in a second pass that cuts it back to K whenever it fills.
//
// Few rows: a row is split over the CTAs of a cluster, whose first CTA joins
// the parts through distributed shared memory: no workspace, and sums in an
// order that depends on the shape and the row's 16-byte alignment alone.
//
// Measured on B200, device time in a stream of calls (floor: the logits at 6.5
// TB/s): 2048 x 131072 bf16 92 us without alternatives, 108 with five (82);
// 4096 x 32000 with five 69 (40); 64 x 131072 f32 with eight 15.4 (5.2); one
// row 9.5.  Many rows are bound by instructions, 9.2 per value (an exponential,
// packed sums, raising, unpacking, maximum) at 64 % of the issue slots, and by
// latency, with 35 % of the warps resident; few rows by the chain of a row's
// beginning and end.  Rows nearly all of one finite mask value overflow the
// lists: 2048 x 131072 404 us.
#include <algorithm>
#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "fw_common.cuh"
#include "fw_kernels.h"

namespace fw {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kUnroll = 4;             // 16-byte loads in flight per thread
constexpr int kListPerWarp = 128;      // places in the list per warp (of eight)
constexpr int kShares = 64;            // values that make a floor
constexpr int kSplitWarps = 8;         // warps of the CTAs that share a row

constexpr int kRankMost = 384;         // candidates ranked by counting
constexpr int kMaxTop = 32;
constexpr int kMaxSplits = 8;          // portable cluster size
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -1.0e4f;     // floor of y: 2^y is 0, and 0 * y stays 0 for y = -inf

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((b & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ float warp_max(float v) { return from_ordered(__reduce_max_sync(kAll, ordered(v))); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// (value descending, index ascending) as one unsigned number; -0 is +0.
__device__ __forceinline__ uint64_t list_key(float v, int e) {
  return (static_cast<uint64_t>(ordered(__fadd_rn(v, 0.0f))) << 32) | static_cast<uint32_t>(~e);
}

// Halfwise maximum of a batch of 16-bit values (a NaN loses).
template <typename R>
__device__ __forceinline__ uint32_t highest2(const uint4 (&v)[kUnroll]) {
  uint32_t h = R::kDead;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) h = R::max2(h, R::max2(R::max2(v[u].x, v[u].y), R::max2(v[u].z, v[u].w)));
  return h;
}

template <int DT>
struct Row;  // N values in 16 bytes
template <>
struct Row<kBf16> {
  static constexpr int N = 8;
  static constexpr uint32_t kDead = 0xff80ff80u;
  __device__ static __forceinline__ void unpack(uint4 v, float* x) {
    x[0] = lo_bf16(v.x), x[1] = hi_bf16(v.x), x[2] = lo_bf16(v.y), x[3] = hi_bf16(v.y);
    x[4] = lo_bf16(v.z), x[5] = hi_bf16(v.z), x[6] = lo_bf16(v.w), x[7] = hi_bf16(v.w);
  }
  __device__ static __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static __forceinline__ float highest(const uint4 (&v)[kUnroll]) {
    const uint32_t h = highest2<Row>(v);
    return fmaxf(lo_bf16(h), hi_bf16(h));
  }
  // v, or the type's lowest value above it
  __device__ static __forceinline__ float at_least(float v) { return bf16_to_f32(f32_to_bf16(fmaxf(v, -3.38e38f))); }
  using Least = uint32_t;
  __device__ static __forceinline__ Least spread(float v) { return (__float_as_uint(v) >> 16) * 0x10001u; }
  __device__ static __forceinline__ uint32_t raise2(uint32_t w, uint32_t low) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(low));
    return r;
  }
  __device__ static __forceinline__ void unpack_raised(uint4 v, Least low, float* x) {
    unpack(make_uint4(raise2(v.x, low), raise2(v.y, low), raise2(v.z, low), raise2(v.w, low)), x);
  }
  __device__ static __forceinline__ float one(const void* p, long long i) {
    return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  }
};
template <>
struct Row<kF16> {
  static constexpr int N = 8;
  static constexpr uint32_t kDead = 0xfc00fc00u;
  __device__ static __forceinline__ void unpack(uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __half2float(__ushort_as_half(static_cast<uint16_t>(w[i])));
      x[2 * i + 1] = __half2float(__ushort_as_half(static_cast<uint16_t>(w[i] >> 16)));
    }
  }
  __device__ static __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static __forceinline__ float highest(const uint4 (&v)[kUnroll]) {
    const uint32_t h = highest2<Row>(v);
    return fmaxf(__half2float(__ushort_as_half(static_cast<uint16_t>(h))),
                 __half2float(__ushort_as_half(static_cast<uint16_t>(h >> 16))));
  }
  __device__ static __forceinline__ float at_least(float v) { return __half2float(__float2half_rn(fmaxf(v, -65504.0f))); }
  using Least = uint32_t;
  __device__ static __forceinline__ Least spread(float v) { return __half_as_ushort(__float2half_rn(v)) * 0x10001u; }
  __device__ static __forceinline__ uint32_t raise2(uint32_t w, uint32_t low) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(low));
    return r;
  }
  __device__ static __forceinline__ void unpack_raised(uint4 v, Least low, float* x) {
    unpack(make_uint4(raise2(v.x, low), raise2(v.y, low), raise2(v.z, low), raise2(v.w, low)), x);
  }
  __device__ static __forceinline__ float one(const void* p, long long i) {
    return __half2float(__ushort_as_half(static_cast<const uint16_t*>(p)[i]));
  }
};
template <>
struct Row<kF32> {
  static constexpr int N = 4;
  static constexpr uint32_t kDead = 0xff800000u;
  __device__ static __forceinline__ void unpack(uint4 v, float* x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  __device__ static __forceinline__ float highest(const uint4 (&v)[kUnroll]) {
    float h = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[N];
      unpack(v[u], x);
#pragma unroll
      for (int i = 0; i < N; ++i) h = fmaxf(h, x[i]);
    }
    return h;
  }
  __device__ static __forceinline__ float at_least(float v) { return fmaxf(v, -3.4e38f); }
  using Least = float;
  __device__ static __forceinline__ Least spread(float v) { return v; }
  __device__ static __forceinline__ void unpack_raised(uint4 v, Least low, float* x) {
    unpack(v, x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = max_nan(x[i], low);
  }
  __device__ static __forceinline__ float one(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
};

// Sums of a part of a row against its maximum m (-inf: nothing yet), without
// the maximum's own term 1 in s.
struct Part {
  float m, s, w;
};
__device__ __forceinline__ Part join(const Part& a, const Part& b, float c) {
  // no finite value: s is 0, or NaN where the part holds one
  if (a.m == -INFINITY) return {b.m, __fadd_rn(a.s, b.s), b.w};
  if (b.m == -INFINITY) return {a.m, __fadd_rn(a.s, b.s), a.w};
  const bool up = a.m < b.m;
  const Part& hi = up ? b : a;
  const Part& lo = up ? a : b;
  const float d = max_nan(__fmul_rn(__fsub_rn(lo.m, hi.m), c), kLowest);
  const float f = ex2(d);
  const float all = __fadd_rn(lo.s, 1.0f);
  return {hi.m, __fadd_rn(hi.s, __fmul_rn(all, f)), __fmaf_rn(__fmaf_rn(d, all, lo.w), f, hi.w)};
}

// W warps work on a row (or a part of one).
template <int W>
struct __align__(16) LogprobSmem {
  static constexpr int kList = W == kSplitWarps ? W * kListPerWarp : 512;
  static constexpr bool kSplit = W == kSplitWarps;
  static constexpr int kHandOn = kList / kMaxSplits;  // keys a part of a split row may hand on
  uint64_t list[kList];       // the warps' candidates, an equal run each; all of it: the careful pass's list
  uint64_t shortlist[kList];  // those of the CTA that reach the floor
  uint64_t merged[kSplit ? kList : 1];  // first CTA of a cluster: those of every part
  uint64_t best[kMaxTop];
  uint4 lane_raw[W][kUnroll];  // one lane's batch, looked at by its warp
  Part part[W];
  Part whole;
  uint32_t share[kShares];  // maxima of the lanes' groups (publish_share)
  uint32_t warp_top[W];     // maxima of the warps, at the end
  float floor;
  int count;  // of list, in the careful pass
  int short_count, merged_count;
  int base;  // where this part's keys go in the first CTA's `merged`
  int found;
};

// The K largest keys of list[0..n) into best, descending; returns how many.
// Called by one whole warp: K rounds of a maximum over the list.
__device__ __forceinline__ int best_of(const uint64_t* list, int n, int K, uint64_t* best, int lane) {
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t mine = 0ull;
    for (int i = lane; i < n; i += 32) {
      const uint64_t v = list[i];
      if (v < last && v > mine) mine = v;
    }
    const uint32_t hi = __reduce_max_sync(kAll, static_cast<uint32_t>(mine >> 32));
    const uint32_t lo =
        __reduce_max_sync(kAll, static_cast<uint32_t>(mine >> 32) == hi ? static_cast<uint32_t>(mine) : 0u);
    last = (static_cast<uint64_t>(hi) << 32) | lo;
    if (last == 0ull) return k;
    if (lane == 0) best[k] = last;
  }
  return K;
}

// The K largest of list[0..n) into sm->best, by the whole CTA between
// barriers of the caller; sets sm->found.  A short list is ranked at once, a
// thread counting the keys above its own (all reads broadcasts); a long one
// takes one warp K rounds.
template <int W>
__device__ __forceinline__ void pick_best(LogprobSmem<W>* sm, const uint64_t* list, int n, int K) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (n <= kRankMost) {
    for (int base = warp * 32; base < n; base += 32 * W) {
      const int i = base + lane;
      const uint64_t key = i < n ? list[i] : 0ull;
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) above += list[j] > key ? 1 : 0;
      if (i < n && above < K) sm->best[above] = key;
    }
    if (threadIdx.x == 0) sm->found = min(n, K);
  } else if (warp == 0) {
    const int found = best_of(list, n, K, sm->best, lane);
    if (lane == 0) sm->found = found;
  }
}

// The K-th largest (K <= 32) of 64 values, two per lane, in every lane: a
// bitonic sort, value i in lane i % 32.
__device__ __forceinline__ uint32_t kth_of_64(uint32_t u, uint32_t v, int K, int lane) {
#pragma unroll
  for (int k = 2; k <= 64; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j == 32) {
        const uint32_t hi = max(u, v), lo = min(u, v);
        u = hi;
        v = lo;
      } else {
        const uint32_t ou = __shfl_xor_sync(kAll, u, j), ov = __shfl_xor_sync(kAll, v, j);
        const bool upper = (lane & j) == 0;
        const bool down_u = (lane & k) == 0, down_v = ((lane + 32) & k) == 0;
        u = upper == down_u ? max(u, ou) : min(u, ou);
        v = upper == down_v ? max(v, ov) : min(v, ov);
      }
    }
  }
  return __shfl_sync(kAll, u, K - 1);
}
// This warp's shares of a floor: the maxima of 64 / W groups of its lanes.
// The K-th largest of all 64 shares is reached by K values at least; a share
// only grows, so that one which is read late still makes a floor.
template <int W>
__device__ __forceinline__ void publish_share(LogprobSmem<W>* sm, float high, int warp, int lane) {
  constexpr int kGroup = W * 32 / kShares;
  uint32_t o = ordered(high);
#pragma unroll
  for (int j = 1; j < kGroup; j <<= 1) o = max(o, __shfl_xor_sync(kAll, o, j));
  if (lane % kGroup == 0) *reinterpret_cast<volatile uint32_t*>(&sm->share[(warp * 32 + lane) / kGroup]) = o;
}
template <int W>
__device__ __forceinline__ float floor_from_shares(const LogprobSmem<W>* sm, int K, int lane) {
  const volatile uint32_t* share = sm->share;
  return from_ordered(kth_of_64(share[lane], share[lane + 32], K, lane));
}

// The careful pass, for row parts with a warp whose candidates overflowed its
// list: the part [v0, v1) over again with one list, cut back to its K best
// whenever the next round might not fit.  The K best end up in sm->best
// (sm->found of them).  All threads.
template <int DT, int W>
__device__ __noinline__ void collect_again(const LogprobArgs& a, long long row, int v0, int v1, LogprobSmem<W>* sm) {
  constexpr int kEach = 8;  // elements of a thread per step
  constexpr int kThreads = 32 * W, kList = LogprobSmem<W>::kList;
  static_assert(kList >= kThreads + kMaxTop, "a round fits beside the K best");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* list = sm->list;
  __syncthreads();
  if (threadIdx.x == 0) sm->count = 0;
  uint64_t last = 0ull;  // key of the K-th best at the last cut
  float floor = -INFINITY;
  auto cut_if_over = [&](int most) {
    __syncthreads();
    const int held = sm->count;
    __syncthreads();  // everyone has read the count that decides
    if (held <= most) return;
    if (warp == 0) {
      const int n = best_of(list, held, a.top_k, sm->best, lane);
      __syncwarp();
      if (lane < n) list[lane] = sm->best[lane];
      if (lane == 0) {
        sm->count = n;
        sm->found = n;
      }
    }
    __syncthreads();
    if (sm->found == a.top_k) {
      last = sm->best[a.top_k - 1];
      floor = fmaxf(floor, from_ordered(static_cast<uint32_t>(last >> 32)));
    }
  };
  for (int base = v0; base < v1; base += kEach * kThreads) {
    float x[kEach];
    float high = -INFINITY;
    bool any = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = base + i * kThreads + threadIdx.x;
      x[i] = e < v1 ? Row<DT>::one(a.logits, row + e) : -INFINITY;
      high = fmaxf(high, x[i]);
      any |= x[i] > -INFINITY && list_key(x[i], e) > last;
    }
    // A step that ends the row may have lanes without values: no floor from it.
    const bool whole = base + kEach * kThreads <= v1;
    if (whole) publish_share(sm, high, warp, lane);
    if (!__syncthreads_or(any)) continue;
    if (whole) floor = fmaxf(floor, floor_from_shares(sm, a.top_k, lane));
#pragma unroll 1
    for (int i = 0; i < kEach; ++i) {
      cut_if_over(kList - kThreads);
      const int e = base + i * kThreads + threadIdx.x;
      float v = -INFINITY;
#pragma unroll
      for (int k = 0; k < kEach; ++k) v = k == i ? x[k] : v;
      const uint64_t key = list_key(v, e);
      if (v > -INFINITY && v >= floor && key > last) list[atomicAdd(&sm->count, 1)] = key;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) sm->found = 0;
  cut_if_over(0);
  __syncthreads();
}

// Two f32 values per 64-bit register, one instruction for both.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack(F2 p, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(p.v));
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

template <int DT, int W>
__global__ void __launch_bounds__(32 * W, 24 / W) k_token_logprobs(const __grid_constant__ LogprobArgs a) {
  using R = Row<DT>;
  constexpr int kThreads = 32 * W, kList = LogprobSmem<W>::kList;
  __shared__ LogprobSmem<W> sm;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x / a.splits, part = blockIdx.x - t * a.splits;
  const long long row = static_cast<long long>(t) * a.stride;
  const int v0 = min(a.vocab, part * a.part_len), v1 = min(a.vocab, v0 + a.part_len);
  const int n = v1 - v0;
  const int K = a.top_k;
  const float c = a.scale;

  // [head scalars][vectors][tail scalars]: vectors start on 16 bytes
  const unsigned char* p = static_cast<const unsigned char*>(a.logits) + (row + v0) * (16 / R::N);
  const int head = min(n, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / (16 / R::N));
  const int nvec = (n - head) / R::N;
  const int first = v0 + head;             // element of vector 0
  const int tail = first + nvec * R::N;    // elements [tail, v1)
  const uint4* vec = reinterpret_cast<const uint4*>(p + static_cast<size_t>(head) * (16 / R::N));

  // A given token's logit is fetched while the row is read.
  int target = -1;
  float target_x = 0.0f;
  if (part == 0 && tid < a.targets_per_row) {
    target = a.targets[static_cast<long long>(t) * a.targets_per_row + tid];
    if (target >= 0 && target < a.vocab) target_x = R::one(a.logits, row + target);
  }

  if (tid == 0) sm.short_count = sm.merged_count = 0;
  // The warp's reference M, its maximum so far.  With mc =
  // fl(M c) the terms are y = fma(z, c, -mc), which is (z - M) c + off for
  // one `off` common to the warp, the rounding of M c: taken out again at the
  // end.  It is half a step of mc at most, so mc is held below 2^24: |off| <=
  // 1/2, and neither 2^off nor a term that counts leaves f32's range.  Values
  // are raised to `least`, far enough below M for 2^y to be 0, so that a
  // masked -inf adds 0 * y = 0.  Where the type has no such number (M near
  // its lowest value, or a high temperature), or M c is larger (rows of far
  // logits, a low temperature, a warp that has seen nothing but a mask of
  // -1e9), `plain` terms are computed as max((z - M) c, kLowest).
  float m = -INFINITY, mc = 0.0f, least = 0.0f;
  bool plain = false;
  F2 s2 = pack(0.0f, 0.0f), w2 = pack(0.0f, 0.0f);  // the lane's sums, even and odd elements
  float seen = -INFINITY;  // the lane's maximum so far
  float floor = INFINITY;                            // candidates are >= floor

  // (S, W) against the exact reference M.
  auto settle = [&]() {
    if (plain || m == -INFINITY) return;
    const float off = __fmaf_rn(m, c, -mc);
    const F2 f = pack(ex2(-off), ex2(-off));
    w2 = mul2(fma2(pack(-off, -off), s2, w2), f);
    s2 = mul2(s2, f);
  };
  // The warp's reference covers `high` (lane maxima).
  auto cover = [&](float high) {
    if (!__any_sync(kAll, high > m)) return;
    const float to = warp_max(high);
    if (m > -INFINITY) {
      settle();
      const float d = max_nan(__fmul_rn(__fsub_rn(m, to), c), kLowest);
      const F2 f = pack(ex2(d), ex2(d));
      w2 = mul2(fma2(pack(d, d), s2, w2), f);
      s2 = mul2(s2, f);
    }
    m = to;
    mc = __fmul_rn(m, c);
    least = R::at_least(__fsub_rn(m, a.depth));
    plain = !(fabsf(mc) < 0x1p24f && __fmul_rn(__fsub_rn(least, m), c) < -1000.0f);
    if (!plain) {  // the sums go on against the rounded reference
      const float off = __fmaf_rn(m, c, -mc);
      const F2 f = pack(ex2(off), ex2(off));
      w2 = mul2(fma2(pack(off, off), s2, w2), f);
      s2 = mul2(s2, f);
    }
  };
  auto add = [&](float x0, float x1) {  // raised to `least` already
    float y0, y1;
    const F2 y = fma2(pack(x0, x1), pack(c, c), pack(-mc, -mc));
    unpack(y, &y0, &y1);
    const F2 e = pack(ex2(y0), ex2(y1));
    s2 = add2(s2, e);
    w2 = fma2(e, y, w2);
  };
  auto add_plain = [&](float x) {
    // (no reference yet: every value is -inf, or NaN)
    const float y = max_nan(__fmul_rn(__fsub_rn(x, m == -INFINITY ? 0.0f : m), c), kLowest);
    const float e = ex2(y);
    s2 = add2(s2, pack(e, 0.0f));
    w2 = fma2(pack(e, 0.0f), pack(y, 0.0f), w2);
  };
  // The warps that have vectors list their candidates in equal runs.
  const int with = max(1, min(W, (nvec + 31) / 32));
  const int run = kList / with;
  uint64_t* list = sm.list + min(warp, with - 1) * run;
  int held = 0;  // candidates of this warp, listed up to `run`
  auto offer = [&](float x, int e) {
    const bool in = x >= floor && x > -INFINITY;
    const unsigned who = __ballot_sync(kAll, in);
    const int at = held + __popc(who & ((1u << lane) - 1u));
    if (in && at < run) list[at] = list_key(x, e);
    held += __popc(who);
  };

  // Head and tail: at most 2 (N - 1) elements, one per lane of warp 0.
  float ragged = -INFINITY;
  int ragged_e = 0;
  if (warp == 0) {
    if (lane < head) ragged_e = v0 + lane;
    else if (lane - head < v1 - tail) ragged_e = tail + lane - head;
    if (lane < head + (v1 - tail)) ragged = R::one(a.logits, row + ragged_e);
    cover(ragged);
    if (lane < head + (v1 - tail)) {
      if (plain || m == -INFINITY) add_plain(ragged);
      else add(max_nan(ragged, least), least);
    }
  }

  const uint4 dead = make_uint4(R::kDead, R::kDead, R::kDead, R::kDead);
  uint4 next[kUnroll];
  auto fetch = [&](int j0) {
    if (j0 + kThreads * kUnroll <= nvec) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) next[u] = ldg_stream(vec + j0 + u * kThreads + tid);
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int j = j0 + u * kThreads + tid;
        next[u] = j < nvec ? ldg_stream(vec + j) : dead;
      }
    }
  };
  fetch(0);
  int raise_at = 1, turn = 0;
  for (int j0 = 0, batch = 1; j0 < nvec; j0 += kThreads * kUnroll, ++batch) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = next[u];
    fetch(j0 + kThreads * kUnroll);
    const float high = R::highest(raw);
    cover(high);
    seen = fmaxf(seen, high);
    if (K > 0) {
      // The floor rises after 1, 2, 4, ... batches, so that each stretch of
      // the row leaves about K candidates; the warps take turns at sorting.
      // Only the first time do they wait for one another.
      if (batch == raise_at) {
        publish_share(&sm, seen, warp, lane);
        if (batch == 1) __syncthreads();
        else __syncwarp();
        if (warp == turn % W) {
          const float f = floor_from_shares(&sm, K, lane);
          if (lane == 0) *reinterpret_cast<volatile float*>(&sm.floor) = f;
        }
        turn += 3;
      }
    }
    if (!plain && m > -INFINITY) {
      const typename R::Least low = R::spread(least);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float x[R::N];
        R::unpack_raised(raw[u], low, x);
#pragma unroll
        for (int i = 0; i < R::N; i += 2) add(x[i], x[i + 1]);
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < kUnroll; ++u) {
        uint4 v = raw[0];
#pragma unroll
        for (int k = 1; k < kUnroll; ++k) v = k == u ? raw[k] : v;
        float x[R::N];
        R::unpack(v, x);
#pragma unroll
        for (int i = 0; i < R::N; ++i) add_plain(x[i]);
      }
    }
    if (K > 0) {
      if (batch == raise_at) {
        if (batch == 1) __syncthreads();
        raise_at *= 2;
      }
      floor = *reinterpret_cast<const volatile float*>(&sm.floor);
      // A lane that has a candidate shows its batch to the warp, an element
      // for each lane.
      for (unsigned who = __ballot_sync(kAll, high >= floor); who != 0u; who &= who - 1u) {
        const int src = __ffs(who) - 1;
        __syncwarp();
        if (lane == src) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) sm.lane_raw[warp][u] = raw[u];
        }
        __syncwarp();
        const float x = lane < kUnroll * R::N ? R::one(sm.lane_raw[warp], lane) : -INFINITY;
        offer(x, first + (j0 + lane / R::N * kThreads + warp * 32 + src) * R::N + lane % R::N);
      }
    }
  }
  seen = fmaxf(seen, ragged);
  if (K > 0 && warp == 0) {
    if (nvec == 0) floor = -INFINITY;
    offer(ragged, ragged_e);
  }
  settle();

  // Join the lanes, then the warps.
  float s_lane, w_lane, s_odd, w_odd;
  unpack(s2, &s_lane, &s_odd);
  unpack(w2, &w_lane, &w_odd);
  s_lane = __fadd_rn(s_lane, s_odd);
  w_lane = __fadd_rn(w_lane, w_odd);
  Part acc;
  acc.m = m;
  acc.s = warp_sum(s_lane);
  if (m > -INFINITY) {
    acc.s = __fsub_rn(acc.s, 1.0f);
    // One value outweighs the others: log S is about their sum, which the 1
    // in the sum of its lane has rounded off.  The warp adds up that lane's
    // values again without the maximum, 1 / 32 of what it has read.
    if (acc.s < 1.0f) {
      const int owner = __ffs(__ballot_sync(kAll, seen == m)) - 1;
      float s = 0.0f, w = 0.0f;
      int more = 0;
      auto add_rest = [&](float x) {
        const float y = max_nan(__fmul_rn(__fsub_rn(x, m), c), kLowest);
        const float e = x == m ? 0.0f : ex2(y);
        more += x == m ? 1 : 0;
        s = __fadd_rn(s, e);
        w = __fmaf_rn(e, y, w);
      };
#pragma unroll 1
      for (int j = warp * 32 + owner + lane * kThreads; j < nvec; j += 32 * kThreads) {
        float x[R::N];
        R::unpack(vec[j], x);
#pragma unroll
        for (int i = 0; i < R::N; ++i) add_rest(x[i]);
      }
      if (lane == owner && ragged > -INFINITY) add_rest(ragged);
      more = static_cast<int>(__reduce_add_sync(kAll, static_cast<unsigned>(more)));
      if (lane != owner) {
        s = __fadd_rn(s, s_lane);
        w = __fadd_rn(w, w_lane);
      }
      acc.s = __fadd_rn(warp_sum(s), static_cast<float>(more - 1));
      w_lane = w;
    }
  }
  acc.w = warp_sum(w_lane);
  if (lane == 0) sm.part[warp] = acc;
  if (K > 0 && LogprobSmem<W>::kSplit && a.splits > 1) {
    const uint32_t top = __reduce_max_sync(kAll, ordered(seen));
    if (lane == 0) sm.warp_top[warp] = top;
  }
  const bool over = __syncthreads_or(held > run);
  const Part none = {-INFINITY, 0.0f, 0.0f};
  // parts[0..n) joined in a fixed order by one warp (n <= 8)
  auto join_all = [&](Part p) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      Part q;
      q.m = __shfl_xor_sync(kAll, p.m, o);
      q.s = __shfl_xor_sync(kAll, p.s, o);
      q.w = __shfl_xor_sync(kAll, p.w, o);
      p = (lane & o) != 0 ? join(q, p, c) : join(p, q, c);
    }
    return p;
  };
  if (warp == W - 1) {
    const Part whole = join_all(lane < W ? sm.part[lane] : none);
    if (lane == 0) sm.whole = whole;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const bool split = LogprobSmem<W>::kSplit && a.splits > 1;
  if (K > 0) {
    if (nvec > 0) floor = *reinterpret_cast<const volatile float*>(&sm.floor);
    if (over) {
      collect_again<DT, W>(a, row, v0, v1, &sm);
      const int found = sm.found;
      held = warp == 0 ? found : 0;
      if (warp == 0 && lane < found) sm.list[lane] = sm.best[lane];
      __syncwarp();
    }
  }
  if (split) {
    cluster.sync();
    if (K > 0) {
      // The K-th largest of all parts' warp maxima (64 at most).
      uint32_t v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (lane + 32 * i) / W;
        v[i] = r < a.splits ? cluster.map_shared_rank(&sm, r)->warp_top[lane % W] : 0u;
      }
      const uint32_t kth = kth_of_64(v[0], v[1], K, lane);
      if (kth != 0u) floor = fmaxf(floor, from_ordered(kth));
    }
    if (part == 0 && warp == W - 1) {
      const Part whole = join_all(lane < a.splits ? cluster.map_shared_rank(&sm, lane)->whole : none);
      __syncwarp();
      if (lane == 0) sm.whole = whole;
    }
  }
  if (K > 0) {
    // This part's candidates that reach the floor.
    const uint64_t least_key = static_cast<uint64_t>(ordered(__fadd_rn(floor, 0.0f))) << 32;
    for (int i = lane; i - lane < held; i += 32) {
      const uint64_t key = i < held ? list[i] : 0ull;
      const bool in = key != 0ull && key >= least_key;
      const unsigned who = __ballot_sync(kAll, in);
      if (who == 0u) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(&sm.short_count, __popc(who));
      at = __shfl_sync(kAll, at, 0) + __popc(who & ((1u << lane) - 1u));
      if (in) sm.shortlist[at] = key;
    }
    __syncthreads();
    int n = sm.short_count;
    const uint64_t* keys = sm.shortlist;
    if (split) {
      // All parts' keys to the first CTA, no more than kHandOn from each.
      if (n > LogprobSmem<W>::kHandOn) {
        pick_best(&sm, keys, n, K);
        __syncthreads();
        keys = sm.best;
        n = sm.found;
      }
      LogprobSmem<W>* to = cluster.map_shared_rank(&sm, 0);
      if (tid == 0) sm.base = n > 0 ? atomicAdd(&to->merged_count, n) : 0;
      __syncthreads();
      if (tid < n) to->merged[sm.base + tid] = keys[tid];
      cluster.sync();
      keys = sm.merged;
      n = sm.merged_count;
    }
    if (part != 0) return;
    pick_best(&sm, keys, n, K);
  } else if (split) {
    cluster.sync();  // the others' sums stay until they have been read
  }
  if (part != 0) return;
  __syncthreads();

  const Part whole = sm.whole;
  const bool bad = !(fabsf(whole.s) <= 3.4e38f);  // a NaN or +inf in the row
  const bool empty = whole.m == -INFINITY;        // every logit is -inf
  const float ln_s = log1pf(whole.s);
  const float nan = __uint_as_float(0x7fc00000u);
  auto logprob = [&](float x) {
    if (bad) return nan;
    if (empty || x == -INFINITY) return -INFINITY;
    // in nats throughout: a representable result does not pass through a
    // larger number (the difference may: it is halved then)
    float y = __fmul_rn(__fsub_rn(x, whole.m), a.inv_temperature);
    if (y == -INFINITY)
      y = __fmul_rn(__fsub_rn(__fmul_rn(x, 0.5f), __fmul_rn(whole.m, 0.5f)), __fmul_rn(a.inv_temperature, 2.0f));
    return __fsub_rn(y, ln_s);
  };
  for (int i = tid; i < a.targets_per_row; i += kThreads) {
    const long long o = static_cast<long long>(t) * a.targets_per_row + i;
    if (i != tid) {
      target = a.targets[o];
      if (target >= 0 && target < a.vocab) target_x = R::one(a.logits, row + target);
    }
    a.logprobs[o] = target < 0 ? 0.0f : target >= a.vocab ? nan : logprob(target_x);
  }
  if (a.entropy != nullptr && tid == kThreads - 1)
    a.entropy[t] = bad ? nan : empty ? 0.0f : __fmaf_rn(-kLn2, __fdiv_rn(whole.w, __fadd_rn(whole.s, 1.0f)), ln_s);
  if (tid < K) {
    const long long o = static_cast<long long>(t) * K + tid;
    const bool there = tid < sm.found && !bad;
    const uint64_t key = there ? sm.best[tid] : 0ull;
    a.top_idx[o] = there ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
    a.top_logprobs[o] = bad ? nan : there ? logprob(from_ordered(static_cast<uint32_t>(key >> 32))) : -INFINITY;
  }
}

constexpr int kNarrowWarps = 2;

template <int DT>
cudaError_t launch_width(const cudaLaunchConfig_t& cfg, const LogprobArgs& a, bool narrow) {
  return narrow ? cudaLaunchKernelEx(&cfg, k_token_logprobs<DT, kNarrowWarps>, a)
                : cudaLaunchKernelEx(&cfg, k_token_logprobs<DT, kSplitWarps>, a);
}

}  // namespace

cudaError_t launch_token_logprobs(LogprobArgs a, cudaStream_t st) {
  DeviceAttrs dev;
  const cudaError_t e = current_device_attrs(&dev);
  if (e != cudaSuccess) return e;
  a.scale = kLog2e * a.inv_temperature;
  a.depth = 20000.0f / a.scale;
  // Few rows: as many parts as the GPU has room for at once (three CTAs of
  // eight warps per SM), of 4096 values at least.
  // Short rows, and many rows of middling length, get two warps each, so that
  // more rows are under way and one's beginning and end hide behind others;
  // long rows keep eight, or too few CTAs would share the end of a launch.
  // Measured with five alternatives, eight against two warps: 4096 x 2000
  // bf16 55 and 19 us, 4096 x 32000 93 and 70 us, 600 x 32000 20.0 and 21.5
  // us, 2048 x 131072 111 and 123 us.
  const int splits = std::max(1, std::min({kMaxSplits, 3 * dev.sms / a.tokens, a.vocab / 4096}));
  a.splits = splits;
  a.part_len = ((a.vocab + splits - 1) / splits + 7) & ~7;
  const bool narrow = splits == 1 && (a.vocab <= 8192 || (a.vocab <= 65536 && a.tokens >= 12 * dev.sms));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.tokens) * splits);
  cfg.blockDim = dim3(32 * (narrow ? kNarrowWarps : kSplitWarps));
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  switch (a.dtype) {
    case kBf16: return launch_width<kBf16>(cfg, a, narrow);
    case kF16: return launch_width<kF16>(cfg, a, narrow);
    default: return launch_width<kF32>(cfg, a, narrow);
  }
}

}  // namespace fw
