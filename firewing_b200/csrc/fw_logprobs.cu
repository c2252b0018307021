// fw_logprobs.cu -- log probabilities of given tokens, entropy and the top
// alternatives of rows of logits (fw_token_logprobs).
//
// For a row z[0..V), c = log2(e) / temperature and a reference M near the
// row's maximum, with y_i = (z_i - M) c:
//   S = sum 2^y_i,  W = sum 2^y_i y_i
//   log p_i = (z_i - M) / temperature - ln S,  H = ln 2 (log2 S - W / S)
// S and W are sums of f32 terms that any part of the row adds up against a
// reference of its own; parts are joined by rescaling.  One pass over the
// row keeps S, W and the candidates for the alternatives.
//
// The reference: each warp takes the maximum of its first batch and changes
// it only when a later value is over it by kSlack powers of two, which f32
// sums stand without loss, so that the loop carries no maximum.
// The alternatives: K values at least are >= `floor`, taken from the first
// batch (the r-th largest of each warp's lane maxima, r = ceil(K / warps),
// and the lowest of these over the warps).  Values under it cost one comparison
// per lane and batch; the few others go to a list in shared memory.  A list
// that overflows (a row of equal values, an ascending row) is made anew in a
// second pass that cuts it back to K whenever it fills.
//
// Few rows: a row is split over the CTAs of a cluster, whose first CTA joins
// the parts through distributed shared memory: no workspace, and sums in an
// order that depends on the shape and the row's 16-byte alignment alone.
#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "fw_common.cuh"
#include "fw_kernels.h"

namespace fw {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kAll = 0xffffffffu;
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnroll = 4;             // 16-byte loads in flight per thread
constexpr int kList = 1024;            // candidates a CTA holds in the fast pass
constexpr int kSlackLog2 = 16;         // how far over its reference (log2) a term may be
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
  __device__ static __forceinline__ float one(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
};

struct Part {  // sums of a part of a row against the reference m (-inf: nothing yet)
  float m, s, w;
};
__device__ __forceinline__ Part join(const Part& a, const Part& b, float c) {
  Part r;
  r.m = fmaxf(a.m, b.m);
  r.s = r.w = 0.0f;
  const Part* p[2] = {&a, &b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (p[i]->m == -INFINITY) {  // no finite value; s is 0, or NaN where the part holds one
      r.s = __fadd_rn(r.s, p[i]->s);
      continue;
    }
    const float d = max_nan(__fmul_rn(__fsub_rn(p[i]->m, r.m), c), kLowest);
    const float f = ex2(d);
    r.s = __fmaf_rn(p[i]->s, f, r.s);
    r.w = __fmaf_rn(__fmaf_rn(d, p[i]->s, p[i]->w), f, r.w);
  }
  return r;
}

struct __align__(16) LogprobSmem {
  uint64_t list[kList];
  uint64_t best[kMaxTop];
  Part part[kWarps];
  Part whole;
  float floor[kWarps];
  int count;
  int found;
};

// The K largest keys of list[0..n) into best, descending; returns how many.
// Called by one whole warp.
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

// The careful pass: the candidates of row part [v0, v1) over again, the list
// cut back to its K best whenever the next round might not fit.  All threads.
template <int DT>
__device__ __noinline__ void collect_again(const LogprobArgs& a, long long row, int v0, int v1, LogprobSmem* sm) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (threadIdx.x == 0) sm->count = kList;  // the list holds this many of the candidates
  uint64_t floor = 0ull;
  for (int base = v0; base < v1; base += kThreads) {
    __syncthreads();
    const int held = sm->count;
    __syncthreads();  // everyone has read the count that decides
    if (held > kList - kThreads) {
      if (warp == 0) {
        const int n = best_of(sm->list, held, a.top_k, sm->best, lane);
        __syncwarp();
        if (lane < n) sm->list[lane] = sm->best[lane];
        if (lane == 0) {
          sm->count = n;
          sm->found = n;
        }
      }
      __syncthreads();
      if (sm->found == a.top_k) floor = sm->best[a.top_k - 1];
    }
    const int e = base + threadIdx.x;
    if (e < v1) {
      const float x = Row<DT>::one(a.logits, row + e);
      const uint64_t key = list_key(x, e);
      if (x > -INFINITY && key > floor) {
        // The list may hold this element from the fast pass already.
        bool there = false;
        for (int i = 0; i < a.top_k; ++i) there |= sm->best[i] == key;
        if (!there) sm->list[atomicAdd(&sm->count, 1)] = key;
      }
    }
  }
  __syncthreads();
}

template <int DT>
__global__ void __launch_bounds__(kThreads) k_token_logprobs(LogprobArgs a) {
  using R = Row<DT>;
  __shared__ LogprobSmem sm;
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

  if (tid == 0) sm.count = 0;
  Part acc = {-INFINITY, 0.0f, 0.0f};
  float m = 0.0f, limit = -INFINITY;  // reference, and the value from which it has to change
  float floor = INFINITY;             // candidates are >= floor

  auto add = [&](float x) {
    const float y = max_nan(__fmul_rn(__fsub_rn(x, m), c), kLowest);
    const float e = ex2(y);
    acc.s = __fadd_rn(acc.s, e);
    acc.w = __fmaf_rn(e, y, acc.w);
  };
  // The warp's reference covers `high` (the warp's values' maximum).
  auto cover = [&](float high) {
    if (__any_sync(kAll, high > limit)) {
      const float to = warp_max(high);
      if (acc.m > -INFINITY) {
        const float d = max_nan(__fmul_rn(__fsub_rn(acc.m, to), c), kLowest);
        const float f = ex2(d);
        acc.w = __fmul_rn(__fmaf_rn(d, acc.s, acc.w), f);
        acc.s = __fmul_rn(acc.s, f);
      }
      acc.m = m = to;
      limit = __fadd_rn(to, a.slack);
    }
  };
  auto offer = [&](float x, int e) {
    if (x >= floor && x > -INFINITY) {
      const int at = atomicAdd(&sm.count, 1);
      if (at < kList) sm.list[at] = list_key(x, e);
    }
  };
  __syncthreads();

  // Head and tail: at most 2 (N - 1) elements, one per lane of warp 0.
  float ragged = -INFINITY;
  int ragged_e = 0;
  if (warp == 0) {
    if (lane < head) ragged_e = v0 + lane;
    else if (lane - head < v1 - tail) ragged_e = tail + lane - head;
    if (lane < head + (v1 - tail)) ragged = R::one(a.logits, row + ragged_e);
    cover(ragged);
    if (lane < head + (v1 - tail)) add(ragged);
  }

  for (int j0 = 0; j0 < nvec; j0 += kThreads * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = j0 + u * kThreads + tid;
      raw[u] = j < nvec ? ldg_stream(vec + j) : make_uint4(R::kDead, R::kDead, R::kDead, R::kDead);
    }
    float high = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[R::N];
      R::unpack(raw[u], x);
#pragma unroll
      for (int i = 0; i < R::N; ++i) high = fmaxf(high, x[i]);
    }
    cover(high);
    if (K > 0) {
      if (j0 == 0) {
        // r-th largest lane maximum of each warp whose lanes all have values
        const int full = min(kWarps, nvec / 32);
        if (full > 0) {
          uint32_t o = ordered(high), r = 0u;
          for (int i = 0; i < (K + full - 1) / full; ++i) {
            r = __reduce_max_sync(kAll, o);
            if (lane == __ffs(__ballot_sync(kAll, o == r)) - 1) o = 0u;
          }
          if (lane == 0) sm.floor[warp] = from_ordered(r);
        }
        __syncthreads();
        floor = full > 0 ? sm.floor[0] : -INFINITY;
        for (int i = 1; i < full; ++i) floor = fminf(floor, sm.floor[i]);
      }
      if (high >= floor) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          float x[R::N];
          R::unpack(raw[u], x);
#pragma unroll
          for (int i = 0; i < R::N; ++i) offer(x[i], first + (j0 + u * kThreads + tid) * R::N + i);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[R::N];
      R::unpack(raw[u], x);
#pragma unroll
      for (int i = 0; i < R::N; ++i) add(x[i]);
    }
  }
  if (K > 0 && warp == 0 && lane < head + (v1 - tail)) {
    if (nvec == 0) floor = -INFINITY;
    offer(ragged, ragged_e);
  }

  // Join the warps.
  acc.s = warp_sum(acc.s);
  acc.w = warp_sum(acc.w);
  if (lane == 0) sm.part[warp] = acc;
  __syncthreads();
  if (K > 0 && sm.count > kList) collect_again<DT>(a, row, v0, v1, &sm);
  if (warp == 0) {
    if (K > 0) {
      const int found = best_of(sm.list, min(sm.count, kList), K, sm.best, lane);
      if (lane == 0) sm.found = found;
    }
    if (lane == 0) {
      Part whole = sm.part[0];
      for (int i = 1; i < kWarps; ++i) whole = join(whole, sm.part[i], c);
      sm.whole = whole;
    }
    __syncwarp();
  }

  // Join the parts of the row in its first CTA.
  if (a.splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0 && warp == 0) {
      if (lane == 0) {
        Part whole = sm.whole;
        for (int r = 1; r < a.splits; ++r) whole = join(whole, cluster.map_shared_rank(&sm, r)->whole, c);
        sm.whole = whole;
      }
      if (K > 0) {
        int total = 0;
        for (int r = 0; r < a.splits; ++r) {
          const LogprobSmem* other = cluster.map_shared_rank(&sm, r);
          const int found = other->found;
          if (lane < found) sm.list[total + lane] = other->best[lane];
          total += found;
        }
        __syncwarp();
        const int found = best_of(sm.list, total, K, sm.best, lane);
        __syncwarp();
        if (lane == 0) sm.found = found;
      }
      __syncwarp();
    }
    cluster.sync();  // the others' shared memory stays until it has been read
    if (part != 0) return;
  }
  __syncthreads();

  const Part whole = sm.whole;
  const bool bad = !(fabsf(whole.s) <= 3.4e38f);  // a NaN or +inf in the row
  const bool empty = whole.s == 0.0f;             // every logit is -inf
  const float log_s = log2f(whole.s);
  const float ln_s = __fmul_rn(log_s, kLn2);
  const float nan = __uint_as_float(0x7fc00000u);
  auto logprob = [&](float x) {
    if (bad) return nan;
    if (empty || x == -INFINITY) return -INFINITY;
    // in nats throughout: a representable result does not pass through a larger number
    return __fsub_rn(__fmul_rn(__fsub_rn(x, whole.m), a.inv_temperature), ln_s);
  };
  for (int i = tid; i < a.targets_per_row; i += kThreads) {
    const long long o = static_cast<long long>(t) * a.targets_per_row + i;
    const int e = a.targets[o];
    a.logprobs[o] = e < 0 ? 0.0f : e >= a.vocab ? nan : logprob(R::one(a.logits, row + e));
  }
  if (a.entropy != nullptr && tid == 0)
    a.entropy[t] = bad ? nan : empty ? 0.0f : __fmul_rn(__fsub_rn(log_s, __fdiv_rn(whole.w, whole.s)), kLn2);
  if (tid < K) {
    const long long o = static_cast<long long>(t) * K + tid;
    const bool there = tid < sm.found && !bad;
    const uint64_t key = there ? sm.best[tid] : 0ull;
    a.top_idx[o] = there ? static_cast<int>(~static_cast<uint32_t>(key)) : -1;
    a.top_logprobs[o] = bad ? nan : there ? logprob(from_ordered(static_cast<uint32_t>(key >> 32))) : -INFINITY;
  }
}

}  // namespace

cudaError_t launch_token_logprobs(LogprobArgs a, cudaStream_t st) {
  DeviceAttrs dev;
  const cudaError_t e = current_device_attrs(&dev);
  if (e != cudaSuccess) return e;
  a.scale = kLog2e * a.inv_temperature;
  a.slack = static_cast<float>(kSlackLog2) / a.scale;
  // Two CTAs per SM at least, while a part has 4096 values.
  int splits = 1;
  while (splits < kMaxSplits && static_cast<long long>(a.tokens) * splits < 2 * dev.sms &&
         a.vocab / (2 * splits) >= 4096)
    splits *= 2;
  a.splits = splits;
  a.part_len = ((a.vocab + splits - 1) / splits + 7) & ~7;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.tokens) * splits);
  cfg.blockDim = dim3(kThreads);
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
    case kBf16: return cudaLaunchKernelEx(&cfg, k_token_logprobs<kBf16>, a);
    case kF16: return cudaLaunchKernelEx(&cfg, k_token_logprobs<kF16>, a);
    default: return cudaLaunchKernelEx(&cfg, k_token_logprobs<kF32>, a);
  }
}

}  // namespace fw
