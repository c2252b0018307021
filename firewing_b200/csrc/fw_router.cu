// fw_router.cu -- routing from a row of logits: softmax or sigmoid scores, a
// balance bias, groups, top-k, renormalised weights (fw_route_scores).
//
// For a token with logits z[0..E):
//   s_e   = softmax(z)_e  or  1 / (1 + exp(-z_e))
//   key_e = s_e + bias_e; without a bias the order of z itself
//   group score = sum of the group's `group_top` (1 or 2) largest keys
//   the `top_groups` best groups, then the K best keys inside them, both by
//   (value descending, index ascending)
//   w_e   = s_e [/ sum of the selected s] * scale
//
// The selection is that of exact arithmetic (64-bit scores), so it does not
// depend on how an exp was rounded: keys are computed in f32 with a known
// error bound, and a row in which two keys that decide something are nearer
// than the bound allows is decided again in 64 bits by the same warp.
//
// One warp per token; lane l holds the experts l, l + 32, ...
#include <cstdint>

#include <cuda_fp16.h>

#include "fw_common.cuh"
#include "fw_kernels.h"

namespace fw {
namespace {

constexpr int kRouteWarps = 4;  // tokens per CTA
constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned kAll = 0xffffffffu;

// Bounds of the f32 scores' errors.  z * log2(e) is off by 2^-23.4 |z log2 e|,
// ex2.approx by 2^-22 relative; for the sigmoid both reach s scaled by
// s (1 - s), with 1 + t, and the quotient adding 2^-23: under 2^-21.8 in
// all.  For the softmax the sum of at most 32 terms per lane and 5 tree
// steps adds 37 * 2^-24 relative: under 2^-18.3 of s.
constexpr float kSigmoidError = 0x1p-20f;          // absolute
constexpr float kSoftmaxError = 0x1p-18f;          // relative to the row's largest score
constexpr float kAddError = 0x1p-23f;              // one f32 addition, relative to its result

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Unsigned order of f32 values; 0 is below every value's (a dead expert).
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((b & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ float load_logit(const void* p, long long i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dtype == kBf16 ? bf16_to_f32(v) : __half2float(__ushort_as_half(v));
}

__device__ __forceinline__ float warp_max(float v) {
  return from_ordered(__reduce_max_sync(kAll, ordered(v)));
}
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// The groups that may be chosen from, as a mask with bit g * lanes set, from
// the keys in `keys` (group g at g * (size + lanes), dead experts -inf).
// 32 / bit_ceil(G) lanes read each group; the padding by `lanes` keeps
// their reads on distinct banks.  *gap: the lowest chosen group's score
// minus the highest other one's (+inf when there is none), *high the
// largest magnitude of the scores compared.
template <typename F>
__device__ __forceinline__ unsigned choose_groups(const F* keys, const RouteScoreArgs& a, int lanes, int lane,
                                                  F* gap, F* high) {
  const F none = static_cast<F>(-INFINITY);
  const int g = lane / lanes, l = lane - g * lanes;
  F m1 = none, m2 = none;
  if (g < a.groups)
    for (int j = l; j < a.group_size; j += lanes) {
      const F v = keys[g * (a.group_size + lanes) + j];
      m2 = fmax(m2, fmin(m1, v));
      m1 = fmax(m1, v);
    }
  for (int o = 1; o < lanes; o <<= 1) {
    const F o1 = __shfl_xor_sync(kAll, m1, o), o2 = __shfl_xor_sync(kAll, m2, o);
    m2 = fmax(fmin(m1, o1), fmax(m2, o2));
    m1 = fmax(m1, o1);
  }
  const F score = (a.group_top == 2 && m2 > none) ? m1 + m2 : m1;
  int before = 0;  // groups that come first
  for (int h = 0; h < a.groups; ++h) {
    const F v = __shfl_sync(kAll, score, h * lanes);
    before += (v > score || (v == score && h < g)) ? 1 : 0;
  }
  const bool chosen = g < a.groups && before < a.top_groups;
  F low = chosen ? score : static_cast<F>(INFINITY);
  F other = (g < a.groups && !chosen) ? score : none;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    low = fmin(low, __shfl_xor_sync(kAll, low, o));
    other = fmax(other, __shfl_xor_sync(kAll, other, o));
  }
  const bool border = other > none;
  *gap = border ? low - other : static_cast<F>(INFINITY);
  *high = border ? fmax(fabs(low), fabs(other)) : static_cast<F>(0);
  return __ballot_sync(kAll, chosen && l == 0);
}

// The selection in 64 bits, for the rows that f32 does not decide: lane k
// returns the k-th selected expert, -1 where there is none.
__device__ __noinline__ int select_in_64_bits(const RouteScoreArgs& a, long long row, int lanes, double* keys,
                                              int lane) {
  const double none = -INFINITY;
  const int E = a.experts;
  double top = none, sum = 0.0;
  if (a.scoring == kScoreSoftmax) {
    for (int e = lane; e < E; e += 32) top = fmax(top, static_cast<double>(load_logit(a.logits, row + e, a.dtype)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, o));
    for (int e = lane; e < E; e += 32) sum += exp(static_cast<double>(load_logit(a.logits, row + e, a.dtype)) - top);
    sum = warp_sum(sum);
  }
  __syncwarp();
  for (int e = lane; e < E; e += 32) {
    const double z = load_logit(a.logits, row + e, a.dtype);
    double key = a.scoring == kScoreSoftmax ? exp(z - top) / sum : 1.0 / (1.0 + exp(-z));
    if (a.bias != nullptr) key += static_cast<double>(a.bias[e]);
    if (z == none) key = none;
    const int g = e / a.group_size;
    keys[e + g * lanes] = key;
  }
  __syncwarp();
  unsigned chosen = kAll;
  if (a.groups > 1) {
    double gap, high;
    chosen = choose_groups<double>(keys, a, lanes, lane, &gap, &high);
  }
  int mine = -1;
  double last = INFINITY;
  int last_e = -1;
  for (int k = 0; k < a.top_k; ++k) {
    double best = none;
    int best_e = E;
    for (int e = lane; e < E; e += 32) {
      const int g = e / a.group_size;
      if (a.groups > 1 && !((chosen >> (g * lanes)) & 1u)) continue;
      const double key = keys[e + g * lanes];
      if (key == none) continue;
      const double v = a.bias != nullptr ? key : static_cast<double>(load_logit(a.logits, row + e, a.dtype));
      if ((v < last || (v == last && e > last_e)) && (v > best || best_e == E)) {
        best = v;
        best_e = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double v = __shfl_xor_sync(kAll, best, o);
      const int e = __shfl_xor_sync(kAll, best_e, o);
      if (e != E && (best_e == E || v > best || (v == best && e < best_e))) {
        best = v;
        best_e = e;
      }
    }
    if (best_e == E) break;
    if (lane == k) mine = best_e;
    last = best;
    last_e = best_e;
  }
  __syncwarp();
  return mine;
}

// NE experts per lane (E <= 32 * NE).
template <int NE>
__global__ void __launch_bounds__(32 * kRouteWarps) k_route_scores(RouteScoreArgs a) {
  extern __shared__ __align__(16) unsigned char route_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x * kRouteWarps + warp;
  if (t >= a.tokens) return;
  const int E = a.experts, K = a.top_k;
  const long long row = static_cast<long long>(t) * a.stride;
  // 64-bit keys of one row per warp; the f32 keys use the same memory
  double* keys64 = reinterpret_cast<double*>(route_smem) + static_cast<size_t>(warp) * (E + 32);
  float* keys = reinterpret_cast<float*>(keys64);
  const bool softmax = a.scoring == kScoreSoftmax;
  const bool biased = a.bias != nullptr;
  const bool grouped = a.groups > 1;
  const int lanes = a.lanes;

  float z[NE];
  bool bad = false;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = i * 32 + lane;
    z[i] = e < E ? load_logit(a.logits, row + e, a.dtype) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    bad |= z[i] != z[i];
    z[i] = __fadd_rn(z[i], 0.0f);  // -0 and +0 are one value
    top = fmaxf(top, z[i]);
  }
  top = warp_max(top);
  bad |= softmax && top == INFINITY;

  // Scores and keys.
  uint32_t order[NE];
  float sum = 0.0f;
  float error = kSigmoidError;
  if (softmax && (biased || grouped || !a.renormalize)) {
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < NE; ++i) sum = __fadd_rn(sum, ex2(__fmul_rn(__fsub_rn(z[i], ref), kLog2e)));
    sum = warp_sum(sum);
    error = __fdividef(kSoftmaxError, sum);
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = i * 32 + lane;
    float key = z[i];
    if (biased || grouped) {
      float s;
      if (softmax) s = __fdividef(ex2(__fmul_rn(__fsub_rn(z[i], top), kLog2e)), sum);
      else s = __fdividef(1.0f, __fadd_rn(1.0f, ex2(__fmul_rn(-z[i], kLog2e))));
      if (biased && e < E) {
        key = __fadd_rn(__fadd_rn(s, a.bias[e]), 0.0f);
        bad |= key != key && z[i] > -INFINITY && !(softmax && top == -INFINITY);
      }
      if (z[i] == -INFINITY) key = -INFINITY;
      if (grouped && e < E) {
        const int g = (e * a.group_inv) >> 20;
        keys[e + g * lanes] = biased || z[i] == -INFINITY ? key : s;
      }
    }
    order[i] = key == -INFINITY ? 0u : ordered(key);
  }
  bad = __any_sync(kAll, bad);

  int mine = -1;  // lane k: the k-th selected expert
  if (!bad) {
    bool again = false;  // f32 does not decide this row
    if (grouped) {
      __syncwarp();
      float gap, high;
      const unsigned chosen = choose_groups<float>(keys, a, lanes, lane, &gap, &high);
      again = !(gap > 2.0f * (a.group_top * error + 3.0f * kAddError * high));
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const int g = ((i * 32 + lane) * a.group_inv) >> 20;
        if (!((chosen >> ((g * lanes) & 31)) & 1u)) order[i] = 0u;  // (an e >= E is dead already)
      }
    }
    // The lane's two best experts after (key, e) = (lo, lo_e).
    uint32_t b1, b2;
    int e1, e2;
    auto scan = [&](uint32_t lo, int lo_e) {
      b1 = b2 = 0u;
      e1 = e2 = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const int e = i * 32 + lane;
        const uint32_t k = order[i];
        const bool after = k < lo || (k == lo && e > lo_e);
        if (after && k > b1) {
          b2 = b1;
          e2 = e1;
          b1 = k;
          e1 = e;
        } else if (after && k > b2) {
          b2 = k;
          e2 = e;
        }
      }
    };
    scan(0xffffffffu, 0x7fffffff);
    bool two = true;
    uint32_t key = 0u;
    // One more than K where the border to the rest has to be looked at.
    const int rounds = biased ? K + 1 : K;
    uint32_t next = 0u;  // the key after the K-th
    for (int k = 0; k < rounds; ++k) {
      const uint32_t m = __reduce_max_sync(kAll, b1);
      if (m == 0u) break;
      const int e = static_cast<int>(__reduce_min_sync(kAll, b1 == m ? static_cast<unsigned>(e1) : 0x7fffffffu));
      if (k == K) {
        next = m;
        if (lane == K) mine = e;  // K = 32 has no such lane: its border counts as near when its key is
        break;
      }
      if (lane == k) {
        key = m;
        mine = e;
      }
      if (lane == (e & 31)) {
        if (two) {
          b1 = b2;
          e1 = e2;
          two = false;
        } else {
          scan(m, e);
          two = true;
        }
      }
    }
    if (biased) {
      // Neighbours in the order have to be further apart than their errors,
      // unless they are the same logit and bias.
      if (lane == K) key = next;
      uint32_t after = __shfl_down_sync(kAll, key, 1);
      const int after_e = __shfl_down_sync(kAll, mine, 1);
      if (lane == 31) after = K == 32 ? next : 0u;
      bool near = false;
      if (lane < K && key != 0u && after != 0u) {
        const float u = from_ordered(key), v = from_ordered(after);
        near = !(__fsub_rn(u, v) > 2.0f * (error + kAddError * fmaxf(fabsf(u), fabsf(v))));
        if (near && key == after && lane < 31)
          near = load_logit(a.logits, row + mine, a.dtype) != load_logit(a.logits, row + after_e, a.dtype) ||
                 a.bias[mine] != a.bias[after_e];
      }
      again |= __any_sync(kAll, near);
      if (lane >= K) mine = -1;
    }
    if (again) {
      __syncwarp();
      mine = select_in_64_bits(a, row, lanes, keys64, lane);
    }
  }

  // Weights of the selected experts: lane k has the k-th.
  float w = 0.0f;
  const bool live = mine >= 0;
  const float zs = live ? load_logit(a.logits, row + mine, a.dtype) : -INFINITY;
  // e^-ref scales numerator and denominator alike, so that scores which
  // all underflow still have their ratios.
  if (softmax) {
    const float ref = a.renormalize ? warp_max(zs) : top;
    if (live) w = expf(__fsub_rn(zs, ref));
    if (!a.renormalize) w = __fdiv_rn(w, sum);
  } else {
    const float ref = a.renormalize ? fminf(warp_max(zs), 0.0f) : 0.0f;
    if (live) w = __fdiv_rn(expf(__fsub_rn(fminf(zs, 0.0f), ref)), __fadd_rn(1.0f, expf(-fabsf(zs))));
  }
  if (a.renormalize) {
    const float total = warp_sum(w);
    w = total > 0.0f ? __fdiv_rn(w, total) : 0.0f;
  }
  w = live ? __fmul_rn(w, a.scale) : 0.0f;
  if (bad) w = __uint_as_float(0x7fc00000u);
  if (lane < K) {
    const long long o = static_cast<long long>(t) * K + lane;
    a.indices[o] = mine;
    a.weights[o] = w;
    if (a.counts != nullptr && live) atomicAdd(a.counts + mine, 1);
  }
}

}  // namespace

cudaError_t launch_route_scores(RouteScoreArgs a, cudaStream_t st) {
  int lanes = 32;
  for (int g = 1; g < a.groups; g <<= 1) lanes >>= 1;
  a.lanes = lanes;
  a.group_size = a.experts / a.groups;
  a.group_inv = (1 << 20) / a.group_size + 1;  // e / group_size = e * inv >> 20 for e, group_size <= 1024
  if (a.counts != nullptr) {
    const cudaError_t e = cudaMemsetAsync(a.counts, 0, sizeof(int32_t) * a.experts, st);
    if (e != cudaSuccess || a.tokens == 0) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.tokens + kRouteWarps - 1) / kRouteWarps);
  cfg.blockDim = dim3(32 * kRouteWarps);
  cfg.dynamicSmemBytes = sizeof(double) * kRouteWarps * (a.experts + 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.experts <= 128) return cudaLaunchKernelEx(&cfg, k_route_scores<4>, a);
  if (a.experts <= 256) return cudaLaunchKernelEx(&cfg, k_route_scores<8>, a);
  if (a.experts <= 512) return cudaLaunchKernelEx(&cfg, k_route_scores<16>, a);
  return cudaLaunchKernelEx(&cfg, k_route_scores<32>, a);
}

}  // namespace fw
