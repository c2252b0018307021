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
//
// Measured on B200, device time in a stream of calls: 8192 x 512 f32 sigmoid
// 8.7 us, with a bias 15.5, with eight groups too 22 (the bytes: 2.7); one
// token 6 to 8.  Bound by instructions, 1800 warp instructions a row in the
// last form at 64 % of the issue slots, and by the latency of dependent ones,
// with 36 % of the warps resident; DRAM is at 7 %.
#include <algorithm>
#include <cstdint>

#include <cuda_fp16.h>

#include "fw_common.cuh"
#include "fw_kernels.h"

namespace fw {
namespace {

constexpr int kRouteWarps = 4;     // tokens per CTA
constexpr int kRouteResident = 7;  // CTAs per SM (half as many with more than 512 experts)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;  // below it a key is dead
constexpr unsigned kAll = 0xffffffffu;

// Bounds of the f32 scores' errors.  z * log2(e) is off by 2^-23.4 |z log2 e|,
// ex2.approx by 2^-22 relative; for the sigmoid both reach s scaled by
// s (1 - s) (at most 1/4, and 0.224 / |z|), 1 + t adds 2^-24 and rcp.approx
// 2^-23: 2.6e-7 in all.  For the softmax the sum of at most 32 terms per lane
// and 5 tree steps adds 37 * 2^-24 relative: under 2^-18.3 of s.
constexpr float kSigmoidError = 0x1.4p-22f;        // absolute, 3e-7
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

template <int DT>
__device__ __forceinline__ float logit_of(const void* p, long long i) {
  if (DT == kF32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return DT == kBf16 ? bf16_to_f32(v) : __half2float(__ushort_as_half(v));
}

// Maximum over the warp; a NaN loses.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// The groups to choose from, as a mask with bit g * lanes set, from the
// groups' scores (group g's in lane g * lanes; -inf: a group of dead experts,
// so that an f32 sum below kLowest is passed as kLowest).  *gap: the lowest chosen
// group's score minus the highest other one's (+inf when there is none),
// *high the largest magnitude of the scores compared.
template <typename F>
__device__ __forceinline__ unsigned rank_groups(F score, const RouteScoreArgs& a, int lanes, int lane, F* gap,
                                                F* high) {
  const F none = static_cast<F>(-INFINITY);
  const int g = lane / lanes;
  const bool owner = g < a.groups && lane == g * lanes;
  int before = 0;  // groups that come first
  for (int h = 0; h < a.groups; ++h) {
    const F v = __shfl_sync(kAll, score, h * lanes);
    before += (v > score || (v == score && h < g)) ? 1 : 0;
  }
  const bool chosen = owner && before < a.top_groups;
  F low = chosen ? score : static_cast<F>(INFINITY);
  F other = owner && !chosen ? score : none;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    low = fmin(low, __shfl_xor_sync(kAll, low, o));
    other = fmax(other, __shfl_xor_sync(kAll, other, o));
  }
  const bool border = other > none;
  *gap = border ? low - other : static_cast<F>(INFINITY);
  *high = border ? fmax(fabs(low), fabs(other)) : static_cast<F>(0);
  return __ballot_sync(kAll, chosen);
}

// The same from the keys in `keys` (group g at g * (size + lanes), dead experts
// -inf).  32 / bit_ceil(G) lanes read each group; the padding by `lanes` keeps
// their reads on distinct banks.
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
  F score = m1;
  if (a.group_top == 2 && m2 > none) score = sizeof(F) == 4 ? fmaxf(m1 + m2, kLowest) : m1 + m2;
  return rank_groups<F>(g < a.groups && l == 0 ? score : none, a, lanes, lane, gap, high);
}

// Shared memory of one warp: f32 or f64 keys of a row (group g shifted by
// g * lanes <= 32), or the candidates being ranked (keys and ids), which may
// stand behind f32 keys.
constexpr int kRanked = 64;
__host__ __device__ inline int warp_doubles(int experts) {
  const int behind = (experts + 33) / 2 + kRanked + kRanked / 2;
  return experts + 32 > behind ? experts + 32 : behind;
}

// Score (and bias) of a logit in 64 bits; top and sum are the softmax's.  One
// exp and one quotient for both kinds: this code runs rarely, and fetching it
// is most of what it costs.
__device__ __forceinline__ double key_in_64_bits(const RouteScoreArgs& a, double z, int e, double top, double sum) {
  const bool softmax = a.scoring == kScoreSoftmax;
  const double x = exp(softmax ? z - top : -z);
  double key = (softmax ? x : 1.0) / (softmax ? sum : 1.0 + x);
  if (a.bias != nullptr) key += static_cast<double>(a.bias[e]);
  return z == -INFINITY ? -INFINITY : key;
}
// Unsigned order of 64-bit values (-0 is +0).
__device__ __forceinline__ uint64_t ordered64(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b ^ ((b >> 63) != 0 ? ~0ull : 1ull << 63);
}
__device__ __noinline__ double softmax_sum_in_64_bits(const void* logits, int dtype, long long row, int E, double top,
                                                      int lane) {
  double sum = 0.0;
  for (int e = lane; e < E; e += 32) sum += exp(static_cast<double>(load_logit(logits, row + e, dtype)) - top);
  return warp_sum(sum);
}
// The groups chosen by 64-bit scores, for a row whose f32 scores leave the
// border open; the row's f32 keys (or logits, whose order is the scores') are
// in `keys` (see choose_groups).  Only the experts that may be among their
// group's two best are looked at, one or two a lane: one such row in thousands
// would otherwise end well after all others (all experts in 64 bits: 6 us).
__device__ __noinline__ unsigned groups_in_64_bits(const RouteScoreArgs& a, long long row, double top, double sum,
                                                   int lanes, float error, const float* keys, int lane) {
  const int g = lane / lanes, l = lane - g * lanes;
  const float* mine = keys + g * (a.group_size + lanes);
  const int size = g < a.groups ? a.group_size : 0;
  float m1 = -INFINITY, m2 = -INFINITY;
  for (int j = l; j < size; j += lanes) {
    const float v = mine[j];
    m2 = fmaxf(m2, fminf(m1, v));
    m1 = fmaxf(m1, v);
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const float o1 = __shfl_xor_sync(kAll, m1, o), o2 = __shfl_xor_sync(kAll, m2, o);
    m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
    m1 = fmaxf(m1, o1);
  }
  float from = a.group_top == 2 && m2 > -INFINITY ? m2 : m1;
  from = fmaxf(__fsub_rn(from, 2.5f * (error + kAddError * fabsf(from))), kLowest);
  uint64_t* spare = reinterpret_cast<uint64_t*>(const_cast<float*>(keys)) + (a.experts + 33) / 2;
  double* exact = reinterpret_cast<double*>(spare);
  int* id = reinterpret_cast<int*>(spare + kRanked);
  int n = 0;
  for (int j = l; j - l < a.group_size; j += lanes) {
    const bool in = j < size && mine[j] >= from;
    const unsigned who = __ballot_sync(kAll, in);
    const int at = n + __popc(who & ((1u << lane) - 1u));
    if (in && at < kRanked) id[at] = g * a.group_size + j;
    n += __popc(who);
  }
  __syncwarp();
  double gap, high, d1 = -INFINITY, d2 = -INFINITY;
  if (n > kRanked) {  // rows of many equal keys
    double* all = reinterpret_cast<double*>(const_cast<float*>(keys));
    for (int e = lane; e < a.experts; e += 32)
      all[e + ((e * a.group_inv) >> 20) * lanes] = key_in_64_bits(a, load_logit(a.logits, row + e, a.dtype), e, top, sum);
    __syncwarp();
    return choose_groups<double>(all, a, lanes, lane, &gap, &high);
  }
#pragma unroll 1
  for (int i = lane; i < n; i += 32)
    exact[i] = key_in_64_bits(a, load_logit(a.logits, row + id[i], a.dtype), id[i], top, sum);
  __syncwarp();
  for (int i = l; i < n; i += lanes) {
    if (((id[i] * a.group_inv) >> 20) != g) continue;
    const double v = exact[i];
    d2 = fmax(d2, fmin(d1, v));
    d1 = fmax(d1, v);
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const double o1 = __shfl_xor_sync(kAll, d1, o), o2 = __shfl_xor_sync(kAll, d2, o);
    d2 = fmax(fmin(d1, o1), fmax(d2, o2));
    d1 = fmax(d1, o1);
  }
  const double score = a.group_top == 2 && d2 > -INFINITY ? d1 + d2 : d1;
  return rank_groups<double>(g < a.groups && l == 0 ? score : -INFINITY, a, lanes, lane, &gap, &high);
}
// Repeated maxima of 64-bit keys, for a row with more near ties than are
// ranked: lane k returns the k-th selected expert, -1 where there is none.
__device__ __noinline__ int select_in_64_bits(const RouteScoreArgs& a, long long row, double top, double sum,
                                              unsigned chosen, int lanes, double* keys, int lane) {
  const int E = a.experts;
  __syncwarp();
  for (int e = lane; e < E; e += 32)
    keys[e] = key_in_64_bits(a, load_logit(a.logits, row + e, a.dtype), e, top, sum);
  __syncwarp();
  int mine = -1;
  double last = INFINITY;
  int last_e = -1;
  for (int k = 0; k < a.top_k; ++k) {
    double best = -INFINITY;
    int best_e = E;
    for (int e = lane; e < E; e += 32) {
      const double v = keys[e];
      if (v == -INFINITY || !((chosen >> ((((e * a.group_inv) >> 20) * lanes) & 31)) & 1u)) continue;
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
// The `n` candidates (ids in id[0..n)) ranked by 64-bit keys: lane k returns
// the k-th.
__device__ __noinline__ int rank_in_64_bits(const RouteScoreArgs& a, long long row, double top, double sum, int n,
                                            uint64_t* keys, int* id, int lane) {
#pragma unroll 1
  for (int i = lane; i < n; i += 32)
    keys[i] = ordered64(key_in_64_bits(a, load_logit(a.logits, row + id[i], a.dtype), id[i], top, sum));
  __syncwarp();
  int mine = -1;
#pragma unroll 1
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    const uint64_t key = i < n ? keys[i] : 0ull;
    const int e = i < n ? id[i] : 0;
    int before = 0;
    for (int j = 0; j < n; ++j) before += (keys[j] > key || (keys[j] == key && id[j] < e)) ? 1 : 0;
    // The candidate of rank k goes to lane k.
    for (int k = 0; k < a.top_k; ++k) {
      const unsigned who = __ballot_sync(kAll, i < n && before == k);
      const int v = __shfl_sync(kAll, e, who != 0u ? __ffs(who) - 1 : 0);
      if (who != 0u && lane == k) mine = v;
    }
  }
  __syncwarp();
  return mine;
}

// Values sorted over the warp, descending: lane k returns the k-th.
__device__ __forceinline__ float sort_lanes(float v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor_sync(kAll, v, j);
      const bool keep_max = ((lane & k) == 0) == ((lane & j) == 0);
      v = keep_max ? fmaxf(v, o) : fminf(v, o);
    }
  }
  return v;
}

// The first `rounds` experts in the order of `keys` (-inf: dead) by repeated
// maxima: lane k gets the k-th one's key and id (id -1 when there is none).
// For the rows whose candidates do not fit the ranking.
template <int NE>
__device__ __noinline__ void select_by_rounds(const float* keys, int rounds, int lane, float* key, int* id) {
  float last = INFINITY;
  int last_e = -1;
  *key = -INFINITY;
  *id = -1;
  for (int k = 0; k < rounds; ++k) {
    float b = -INFINITY;
    int be = 0x7fffffff;
    for (int i = 0; i < NE; ++i) {
      const int e = i * 32 + lane;
      const float v = keys[i];
      if ((v < last || (v == last && e > last_e)) && v > b) {
        b = v;
        be = e;
      }
    }
    const float m = warp_max(b);
    if (m == -INFINITY) break;
    const int e = static_cast<int>(__reduce_min_sync(kAll, b == m ? static_cast<unsigned>(be) : 0x7fffffffu));
    if (lane == k) {
      *key = m;
      *id = e;
    }
    last = m;
    last_e = e;
  }
}

// NE experts per lane (E <= 32 * NE), logits of type DT.  A warp takes the
// rows warp, warp + warps, ....  EVEN: E = 32 * NE and the groups, if any, are made of whole
// runs of 32 experts, so that a lane has as many of each: their scores then
// take two reductions each and no shared memory.
template <int NE, int DT, bool EVEN>
__global__ void __launch_bounds__(32 * kRouteWarps, NE <= 16 ? kRouteResident : kRouteResident / 2)
    k_route_scores(const __grid_constant__ RouteScoreArgs a) {
  extern __shared__ __align__(16) unsigned char route_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = EVEN ? 32 * NE : a.experts, K = a.top_k;
  double* keys64 = reinterpret_cast<double*>(route_smem) + static_cast<size_t>(warp) * warp_doubles(E);
  float* keys = reinterpret_cast<float*>(keys64);
  uint64_t* ranked = reinterpret_cast<uint64_t*>(keys64);
  int* loads = reinterpret_cast<int*>(reinterpret_cast<double*>(route_smem) + kRouteWarps * warp_doubles(E));
  const bool softmax = a.scoring == kScoreSoftmax;
  const bool biased = a.bias != nullptr;
  const bool grouped = a.groups > 1;
  const int lanes = a.lanes;
  const int shift = EVEN ? a.run_shift : 0;  // log2 of a group's runs of 32 experts
  const int first = blockIdx.x * kRouteWarps + warp, step = gridDim.x * kRouteWarps;
  if (a.counts != nullptr) {
    for (int e = threadIdx.x; e < E; e += blockDim.x) loads[e] = 0;
    __syncthreads();
  }
  pdl_wait();
  pdl_launch_dependents();

  float* biases = reinterpret_cast<float*>(loads + E);
  bool nan_bias = false;
  if (biased) {
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
      const float v = a.bias[e];
      biases[e] = v;
      nan_bias |= v != v;
    }
    nan_bias = __syncthreads_or(nan_bias);
  }
  // A group's score may be small and its two keys large, with their error: of
  // opposite signs they take away from each other no more than the positive
  // one, at most the largest bias + 1, or the other one, at most the size of
  // the lowest bias that is a number.
  __shared__ float bias_most[kRouteWarps], bias_least[kRouteWarps];
  if (biased && grouped && a.group_top == 2) {
    float most = -INFINITY, least = INFINITY;
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
      most = fmaxf(most, biases[e]);
      if (biases[e] > -INFINITY) least = fminf(least, biases[e]);
    }
    most = warp_max(most);
    least = -warp_max(-least);
    if (lane == 0) {
      bias_most[warp] = most;
      bias_least[warp] = least;
    }
    __syncthreads();
  }

  for (int t = first; t < a.tokens; t += step) {
    const long long row = t * a.stride;
    float z[NE];
    bool bad = false;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      z[i] = EVEN || i * 32 + lane < E ? logit_of<DT>(a.logits, row + lane + i * 32) : -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      bad |= z[i] != z[i];
      z[i] = __fadd_rn(z[i], 0.0f);  // -0 and +0 are one value
      top = fmaxf(top, z[i]);
    }
    top = warp_max(top);
    bad |= softmax && top == INFINITY;

    // Scores and keys (-inf: out of the question).
    float key[NE];
    float sum = 0.0f, inv_sum = 0.0f;
    float error = kSigmoidError;
    const float ref = top == -INFINITY ? 0.0f : top;
    if (softmax && (biased || grouped || !a.renormalize)) {
#pragma unroll
      for (int i = 0; i < NE; ++i) sum = __fadd_rn(sum, ex2(__fmul_rn(__fsub_rn(z[i], ref), kLog2e)));
      sum = warp_sum(sum);
      inv_sum = rcp(sum);
      error = __fmul_rn(kSoftmaxError, inv_sum);
    }
    __syncwarp();  // the previous row is done with the shared memory
    float score = -INFINITY;            // EVEN: lane g's is group g's
    float m1 = -INFINITY, m2 = -INFINITY;  // the lane's two largest of the group being passed
    if (biased || grouped) {
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        float s;
        if (softmax) s = __fmul_rn(ex2(__fmul_rn(__fsub_rn(z[i], ref), kLog2e)), inv_sum);
        else s = rcp(__fadd_rn(1.0f, ex2(__fmul_rn(z[i], -kLog2e))));
        float k = s;
        if (biased) {
          k = __fadd_rn(__fadd_rn(s, EVEN || i * 32 + lane < E ? biases[i * 32 + lane] : 0.0f), 0.0f);
          if (nan_bias) bad |= k != k && z[i] > -INFINITY;
        }
        if (z[i] == -INFINITY) k = -INFINITY;
        key[i] = biased ? k : z[i];
        if (grouped) {
          if (EVEN) {
            m2 = fmaxf(m2, fminf(m1, k));
            m1 = fmaxf(m1, k);
            if ((((i + 1) >> shift) << shift) == i + 1) {
              const float best = warp_max(m1);
              float value = best;
              if (a.group_top == 2) {
                const unsigned who = __ballot_sync(kAll, m1 == best);
                const float second = warp_max(lane == __ffs(who) - 1 ? m2 : m1);
                if (second > -INFINITY) value = fmaxf(__fadd_rn(best, second), kLowest);
              }
              if (lane == i >> shift) score = value;
              m1 = m2 = -INFINITY;
            }
          } else if (i * 32 + lane < E) {
            const int e = i * 32 + lane;
            keys[e + ((e * a.group_inv) >> 20) * lanes] = k;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NE; ++i) key[i] = z[i];
    }
    bad = __any_sync(kAll, bad);

    int mine = -1;  // lane k: the k-th selected expert
    if (!bad && top > -INFINITY) {
      unsigned chosen = kAll;           // bit g * lanes (bit g where `narrow`): group g stays
      bool narrow = false;
      double top64 = top, sum64 = 0.0;  // the softmax in 64 bits, where it is needed
      if (grouped) {
        __syncwarp();
        float gap, high;
        int spread = lanes;
        if (EVEN) {
          chosen = rank_groups<float>(score, a, 1, lane, &gap, &high);
          spread = 1;  // (widened where the 64-bit functions need it)
        } else {
          chosen = choose_groups<float>(keys, a, lanes, lane, &gap, &high);
        }
        if (biased && a.group_top == 2) {
          float most = bias_most[0], least = bias_least[0];
#pragma unroll
          for (int i = 1; i < kRouteWarps; ++i) {
            most = fmaxf(most, bias_most[i]);
            least = fminf(least, bias_least[i]);
          }
          high = __fmaf_rn(2.0f, fmaxf(fminf(__fadd_rn(most, 1.0f), -least), 0.0f), high);
        }
        if (!(gap > 2.0f * (a.group_top * error + 3.0f * kAddError * high))) {
          if (softmax) sum64 = softmax_sum_in_64_bits(a.logits, DT, row, E, top64, lane);
          if (EVEN) {
#pragma unroll
            for (int i = 0; i < NE; ++i) keys[i * 32 + lane + (i >> shift) * lanes] = key[i];
          }
          __syncwarp();
          chosen = groups_in_64_bits(a, row, top64, sum64, lanes, error, keys, lane);
          __syncwarp();
          spread = lanes;
        }
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          const int g = EVEN ? i >> shift : ((i * 32 + lane) * a.group_inv) >> 20;
          if (!((chosen >> ((g * spread) & 31)) & 1u)) key[i] = -INFINITY;  // (an e >= E is dead already)
        }
        narrow = spread != lanes;
      }
      float lane_best = -INFINITY;
#pragma unroll
      for (int i = 0; i < NE; ++i) lane_best = fmaxf(lane_best, key[i]);
      // K lanes at least reach the K-th largest lane maximum: candidates are
      // the keys from there on.
      float floor;
      if (K <= 16) {
        floor = lane_best;
        for (int k = 1;; ++k) {
          const float best = warp_max(floor);
          if (k == K) {
            floor = best;
            break;
          }
          if (floor == best) floor = -INFINITY;  // (equal maxima go together: the floor is lower then)
        }
      } else {
        floor = __shfl_sync(kAll, sort_lanes(lane_best, lane), K - 1);
      }
      floor = fmaxf(floor, kLowest);
      // How many candidates the lane has from `from` on, and where they go.
      auto place = [&](float from, int* n) {
        int mine_here = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) mine_here += key[i] >= from ? 1 : 0;
        int before = mine_here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(kAll, before, o);
          if (lane >= o) before += v;
        }
        *n = __shfl_sync(kAll, before, 31);
        return before - mine_here;
      };
      int n;
      int at = place(floor, &n);
      float my_key = -INFINITY, after = -INFINITY;  // lane k: the k-th key, and the one behind it
      int after_e = -1;
      __syncwarp();
      if (n <= kRanked) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
          if (key[i] >= floor)
            ranked[at++] = (static_cast<uint64_t>(ordered(key[i])) << 32) | static_cast<uint32_t>(~(i * 32 + lane));
        __syncwarp();
        // Rank each candidate by the number of those before it.
        const uint64_t u = lane < n ? ranked[lane] : 0ull, v = lane + 32 < n ? ranked[lane + 32] : 0ull;
        int ru = 0, rv = 0;
        if (n <= 32) {
#pragma unroll 4
          for (int j = 0; j < n; ++j) ru += ranked[j] > u ? 1 : 0;
        } else {
          for (int j = 0; j < n; ++j) {
            const uint64_t o = ranked[j];
            ru += o > u ? 1 : 0;
            rv += o > v ? 1 : 0;
          }
        }
        __syncwarp();
        if (lane < n) ranked[ru] = u;
        if (lane + 32 < n) ranked[rv] = v;
        __syncwarp();
        if (lane < n) {
          my_key = from_ordered(static_cast<uint32_t>(ranked[lane] >> 32));
          mine = static_cast<int>(~static_cast<uint32_t>(ranked[lane]));
        }
        if (lane + 1 < n) {
          after = from_ordered(static_cast<uint32_t>(ranked[lane + 1] >> 32));
          after_e = static_cast<int>(~static_cast<uint32_t>(ranked[lane + 1]));
        }
        __syncwarp();
      } else {
        float copy[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) copy[i] = key[i];
        select_by_rounds<NE>(copy, 32, lane, &my_key, &mine);
        after = __shfl_down_sync(kAll, my_key, 1);
        after_e = __shfl_down_sync(kAll, mine, 1);
        if (lane == 31) {  // the key behind has no lane and counts as near
          after = my_key;
          after_e = -1;
        }
      }
      if (biased) {
        // Neighbours in the order have to be further apart than their errors,
        // unless they are the same logit and bias: the first K and the one
        // behind them, and where those at the border are the same, all
        // that follow as near.
        const auto is_close = [&](float behind) {
          return behind > -INFINITY &&
                 !(__fsub_rn(my_key, behind) > 2.0f * (error + kAddError * fmaxf(fabsf(my_key), fabsf(behind))));
        };
        const bool close = is_close(after);
        bool other = close;
        if (close && my_key == after && after_e >= 0)
          other = logit_of<DT>(a.logits, row + mine) != logit_of<DT>(a.logits, row + after_e) ||
                  a.bias[mine] != a.bias[after_e];
        const unsigned apart = ~(__ballot_sync(kAll, close) >> (K - 1));
        const int end = K - 1 + (apart != 0u ? __ffs(apart) - 1 : 32);  // the last of them
        bool near = other && lane < max(end, K);
        if (end > 31) near = true;  // (they pass the lanes)
        // The best key that is no candidate stands behind the last one.
        if (n <= K || end == n - 1) {
          float below = -INFINITY;
#pragma unroll
          for (int i = 0; i < NE; ++i) below = fmaxf(below, key[i] < floor ? key[i] : -INFINITY);
          below = warp_max(below);
          if (lane == n - 1) near |= is_close(below);
        }
        if (__any_sync(kAll, near)) {
          if (softmax && sum64 == 0.0) sum64 = softmax_sum_in_64_bits(a.logits, DT, row, E, top64, lane);
          // Every expert that may be among the K best: down to the K-th key
          // less both errors.
          const float kth = __shfl_sync(kAll, my_key, K - 1);
          const float low = __fsub_rn(kth, 2.5f * (error + kAddError * fabsf(kth)));
          const float from = fmaxf(low, kLowest);  // (no K-th key: everything)
          __syncwarp();
          int* id = reinterpret_cast<int*>(keys64 + kRanked);
          at = place(from, &n);
          if (n <= kRanked) {
#pragma unroll
            for (int i = 0; i < NE; ++i)
              if (key[i] >= from) id[at++] = i * 32 + lane;
            __syncwarp();
            mine = rank_in_64_bits(a, row, top64, sum64, n, ranked, id, lane);
          } else {
            if (narrow) {
              unsigned wide = 0u;
              for (int g = 0; g < a.groups; ++g) wide |= ((chosen >> g) & 1u) << (g * lanes);
              chosen = wide;
            }
            mine = select_in_64_bits(a, row, top64, sum64, chosen, lanes, keys64, lane);
          }
        }
      }
      if (lane >= K) mine = -1;
    }

    // Weights of the selected experts: lane k has the k-th.
    float w = 0.0f;
    const bool live = mine >= 0;
    const float zs = live ? logit_of<DT>(a.logits, row + mine) : -INFINITY;
    // e^-ref scales numerator and denominator alike, so that scores which
    // all underflow still have their ratios.
    if (softmax) {
      const float high = a.renormalize ? warp_max(zs) : top;
      if (live) w = expf(__fsub_rn(zs, high));
      if (!a.renormalize) w = __fdividef(w, sum);
    } else {
      const float high = a.renormalize ? fminf(warp_max(zs), 0.0f) : 0.0f;
      if (live) w = __fdividef(expf(__fsub_rn(fminf(zs, 0.0f), high)), __fadd_rn(1.0f, expf(-fabsf(zs))));
    }
    if (a.renormalize) {
      const float total = warp_sum(w);
      w = total > 0.0f ? __fdividef(w, total) : 0.0f;
    }
    w = live ? __fmul_rn(w, a.scale) : 0.0f;
    if (bad) w = __uint_as_float(0x7fc00000u);
    if (lane < K) {
      const long long o = static_cast<long long>(t) * K + lane;
      a.indices[o] = mine;
      a.weights[o] = w;
      if (a.counts != nullptr && live) atomicAdd(loads + mine, 1);
    }
  }
  if (a.counts != nullptr) {
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x)
      if (loads[e] != 0) atomicAdd(a.counts + e, loads[e]);
  }
}

__global__ void k_clear_counts(int32_t* counts, int experts) {
  pdl_wait();
  pdl_launch_dependents();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[e] = 0;
}

template <int NE, bool EVEN>
cudaError_t launch_even(const cudaLaunchConfig_t& cfg, const RouteScoreArgs& a) {
  switch (a.dtype) {
    case kBf16: return cudaLaunchKernelEx(&cfg, k_route_scores<NE, kBf16, EVEN>, a);
    case kF16: return cudaLaunchKernelEx(&cfg, k_route_scores<NE, kF16, EVEN>, a);
    default: return cudaLaunchKernelEx(&cfg, k_route_scores<NE, kF32, EVEN>, a);
  }
}
template <int NE>
cudaError_t launch_ne(const cudaLaunchConfig_t& cfg, const RouteScoreArgs& a) {
  const bool even = a.experts == 32 * NE && (a.groups == 1 || a.group_size % 32 == 0);
  return even ? launch_even<NE, true>(cfg, a) : launch_even<NE, false>(cfg, a);
}

}  // namespace

cudaError_t launch_route_scores(RouteScoreArgs a, cudaStream_t st) {
  int lanes = 32;
  for (int g = 1; g < a.groups; g <<= 1) lanes >>= 1;
  a.lanes = lanes;
  a.group_size = a.experts / a.groups;
  a.run_shift = 0;
  while ((64 << a.run_shift) <= a.group_size) ++a.run_shift;
  a.group_inv = (1 << 20) / a.group_size + 1;  // e / group_size = e * inv >> 20 for e, group_size <= 1024
  cudaLaunchConfig_t cfg = {};
  // Every row a warp of its own while the GPU has room for all of them, then
  // a share of the rows each.  A row is a long chain of dependent steps, so
  // resident warps count: 8192 rows of 512 experts took 11.4 us with 16 per SM,
  // 8.7 us with 28 (sigmoid without bias or groups).  Fetching the next row
  // early, or keeping the bias in registers, costs more warps than it gains.
  DeviceAttrs dev;
  const cudaError_t de = current_device_attrs(&dev);
  if (de != cudaSuccess) return de;
  cfg.gridDim = dim3(std::min((a.tokens + kRouteWarps - 1) / kRouteWarps, dev.sms * kRouteResident));
  cfg.blockDim = dim3(32 * kRouteWarps);
  cfg.dynamicSmemBytes = sizeof(double) * kRouteWarps * warp_doubles(a.experts) + 2 * sizeof(int) * a.experts;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.counts != nullptr) {
    // A kernel of our own, so that the next one's launch overlaps it.
    cudaLaunchConfig_t clear = cfg;
    clear.gridDim = dim3(1);
    clear.blockDim = dim3(256);
    clear.dynamicSmemBytes = 0;
    const cudaError_t e = cudaLaunchKernelEx(&clear, k_clear_counts, a.counts, a.experts);
    if (e != cudaSuccess || a.tokens == 0) return e;
  }
  if (a.experts <= 128) return launch_ne<4>(cfg, a);
  if (a.experts <= 256) return launch_ne<8>(cfg, a);
  if (a.experts <= 512) return launch_ne<16>(cfg, a);
  return launch_ne<32>(cfg, a);
}

}  // namespace fw
