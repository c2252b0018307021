// fw_linear.cu -- y = act(x w^T + bias) + residual (fw_linear_epilogue).
//
// x [T][K], w [N][K], bf16 or f16; sums in f32; bias, activation and residual
// in f32 on the accumulator; one rounding to y's type.
//
// k_linear_pair: many tokens.  Two CTAs on one 256 x 256 tile (see there).
// k_linear_mma: the others on the tensor cores.  One operand is the M side
//   (P, 128 rows per tile), the other the N side (Q, bn rows per tile, a
//   multiple of 16 up to 256); both are K-major, staged 64 columns at a time
//   in the 128-byte swizzled layout.
//     warp 0      producer: TMA loads of both tiles into a ring
//     warp 1      tcgen05.mma kind::f16 into one of two TMEM accumulators
//                 (tiles shared by a cluster: one)
//     warps 2-9   epilogue, two sets of four (set s takes the 32-column
//                 groups s, s + 2, ...)
//     Where TMA cannot read an operand (a row stride or base that is no
//     multiple of 16 bytes) warps 2-5 are the epilogue and warps 6-21
//     loaders, which bring the rows into shared memory by cp.async, realign
//     them in registers and write the same layout
//   Few tokens: w is the M side and the K range is split over the CTAs of a
//   cluster, which exchange their partial tiles through distributed shared
//   memory and add them in rank order (no workspace, repeatable sums).
// k_linear_rows: one to a few tokens on the CUDA cores, a warp (or several)
//   per weight row: the weights' bytes are the work, and there is no
//   pipeline to fill.
//
// Measured on B200, device time in a stream of calls (floor: the operands'
// bytes at 6.5 TB/s, or the products at 1.66 PFLOP/s):
//   8192 x 8192 x 2048 bf16, bias, GELU (tanh)  176-184 us  (165): the MMAs
//   8192 x 8192 x 8192 bf16                        682 us  (661)
//   8192 x 8192 x 2048 bf16, f32 out           242-257 us  (165): the f32
//     outputs' way out of registers, which the next tile hides in part
//   4096 x 2048 x 8192 bf16, residual          107-124 us   (83): 128 tiles
//     in two waves of 74 pairs
//   64 x 8192 x 2048 bf16, bias, SiLU             12.2 us  (5.4): the first
//     loads' way, 16 blocks of a CTA, the epilogue, one after the other (11.4
//     where L2 keeps some of the weights)
//   333 x 1001 x 1999 f16, bias, GELU, residual   15.7 us  (1.0): the loaders
//     (29 to 32 bytes per ns and SM), the joint, code that runs once
//   8000 x 8001 x 2001 f16                         886 us  (154): the loaders
//   1 x 512 x 2048 bf16                            3.0 us  (0.3): a launch and
//     two trips to memory
//
// Every wait is for one step and bounded (2 s of globaltimer, or what
// fw_primitive_set_wait_limit says); on expiry the CTA records a time-out, lets
// its copies and MMAs drain (bounded), frees its TMEM and exits;
// fw_primitive_status reports it.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <mutex>

#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include "fw_common.cuh"
#include "fw_kernels.h"

namespace fw {
namespace {

constexpr int kBM = 128;                  // M-side rows per tile
constexpr int kBK = 64;                   // columns per stage (one 128-byte swizzle atom)
constexpr int kABytes = kBM * kBK * 2;    // 16 KB
constexpr int kMaxStages = 8;
constexpr int kEpiWarps = 8;
constexpr int kLoadWarps = 16;
// The loaders are two groups that take turns at stages: what a warp waits for
// in a stage (its words, the slot, the fence) would otherwise bound it.
constexpr int kLoadGroups = 2;
constexpr int kGroupWarps = kLoadWarps / kLoadGroups;
constexpr int kWarpRows = 32;              // rows of a stage that a loader warp fills, at most
constexpr int kLoadBn = 128;               // N tiles are this wide at most
constexpr int kAhead = 1;                  // stages of its own that a group fetches ahead
constexpr int kRawBytes = kWarpRows * 144; // a warp's words of a stage
constexpr int kLoadStages = 2;             // operand stages beside them
constexpr int kRawTotal = kLoadWarps * (kAhead + 1) * kRawBytes;
// Warps of a group for the P rows, so that both sides' warps have about as
// many rows; the others serve the Q rows.
__host__ __device__ constexpr int p_warps(int bn) { return (kGroupWarps * kBM + (kBM + bn) / 2) / (kBM + bn); }
constexpr bool loaders_hold(int bn) {
  return bn > kLoadBn || (p_warps(bn) < kGroupWarps && p_warps(bn) * kWarpRows >= kBM &&
                          (kGroupWarps - p_warps(bn)) * kWarpRows >= bn && loaders_hold(bn + 16));
}
static_assert(loaders_hold(16), "every row of a stage has a loader");
constexpr int kMmaThreads = 32 * (2 + kEpiWarps);
// With loaders half the epilogue warps: N tiles are narrow then.
constexpr int kLoaderEpiWarps = 4;
constexpr int kLoaderThreads = 32 * (2 + kLoaderEpiWarps + kLoadWarps);
// Stages per accumulation for f32 outputs: the tensor cores truncate, which
// left K = 8192 1.4e-6 off in one accumulation, 4.4e-7 in pieces of 512 columns
// added in registers (an f32 product on the CUDA cores: 9.6e-7).
constexpr int kChunk = 8;
constexpr int kMostSmem = 227 * 1024;
constexpr unsigned kAll = 0xffffffffu;

__device__ int g_status;  // first time-out of this library's linear kernels on the device

// ---- tcgen05 / TMA ----------------------------------------------------------------

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major operand, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// kind::f16, both operands bf16 or both f16, K-major, f32 accumulator, M x N.
__device__ __forceinline__ uint32_t idesc_f16(int m, int n, bool bf16) {
  const uint32_t type = bf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// The same for a pair of CTAs (issued by the even one): M = 256, A rows and N
// rows split over the two CTAs' shared memory at the same offsets, D in both
// CTAs' TMEM; the commit arrives at the same barrier of both.
__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// A load into this CTA's shared memory that completes on a barrier of the
// pair (`bar`: its shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
// One lane of a converged warp, always the same.  The producer and MMA warps
// run their loops with all lanes, so that addresses and descriptors stay in
// uniform registers, and issue with the elected one.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 32 (16) consecutive f32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t saddr, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

// ---- epilogue arithmetic -------------------------------------------------------------

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// Two f32 values per 64-bit register, one instruction for both.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 pack(float a) { return pack(a, a); }
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
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float relu(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
  return r;
}
// x/2 (1 + erf(x / sqrt 2)) = max(x, 0) - |x|/2 erfc(|x| / sqrt 2) per half,
// with erfc(z) = t 2^(-z^2 log2 e + g(t)), t = 1 / (1 + z / 2), the form of
// erfcc in Press et al., Numerical Recipes: t takes z >= 0 to (0, 1], where
// log2(erfc(z) exp(z^2) / t) is smooth.  g is its least squares fit at the
// Chebyshev points, degree 9, made for this file: erfc to 1.1e-7 relative for
// every z.  In f32 the exponent's three roundings come on top, 3 2^-24 of its
// size in nats, x^2 / 2: of a result 4e-7 near 0, 8e-6 at x = -12.
__device__ __forceinline__ F2 gelu2(F2 v) {
  constexpr float g[10] = {-1.82574821f, 1.44272923f,  0.539700329f, 0.139632389f,  -0.268766135f,
                           0.402343214f, -1.63778341f, 2.14749932f,  -1.18612599f, 0.246519342f};
  float x, y;
  unpack(v, &x, &y);
  // (an infinite size would meet erfc = 0 in a product)
  const F2 size = pack(fminf(fabsf(x), 1e30f), fminf(fabsf(y), 1e30f));
  float t0, t1;
  unpack(fma2(size, pack(0.35355339059327376f), pack(1.0f)), &t0, &t1);
  const F2 t = pack(rcp(t0), rcp(t1));
  F2 p = pack(g[9]);
#pragma unroll
  for (int i = 8; i >= 0; --i) p = fma2(p, t, pack(g[i]));
  p = fma2(mul2(v, v), pack(-0.5f * kLog2e), p);
  unpack(p, &t0, &t1);
  const F2 e = mul2(mul2(t, pack(ex2(t0), ex2(t1))), mul2(size, pack(-0.5f)));
  return add2(pack(relu(x), relu(y)), e);
}

__device__ __forceinline__ float load_f32(const void* p, long long i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dtype == kBf16 ? bf16_to_f32(v) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ void store_f32(void* p, long long i, int dtype, float v) {
  if (dtype == kF32) static_cast<float*>(p)[i] = v;
  else if (dtype == kBf16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<uint16_t*>(p)[i] = __half_as_ushort(__float2half_rn(v));
}
// Two values rounded to a 16-bit type, the first in the low half.
__device__ __forceinline__ uint32_t pack2(int dtype, float lo, float hi) {
  uint32_t r;
  if (dtype == kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void unpack2(int dtype, uint32_t w, float* lo, float* hi) {
  if (dtype == kBf16) {
    *lo = lo_bf16(w);
    *hi = hi_bf16(w);
  } else {
    *lo = __half2float(__ushort_as_half(static_cast<uint16_t>(w)));
    *hi = __half2float(__ushort_as_half(static_cast<uint16_t>(w >> 16)));
  }
}
// x / (1 + 2^z) per half: 1 + 2^z = inf gives 0.
__device__ __forceinline__ F2 gate2(F2 x, F2 z) {
  float z0, z1;
  unpack(z, &z0, &z1);
  unpack(add2(pack(ex2(z0), ex2(z1)), pack(1.0f)), &z0, &z1);
  return mul2(x, pack(rcp(z0), rcp(z1)));
}
// -inf as the lowest finite value, which a gate of 0 makes 0, the limit.
__device__ __forceinline__ F2 finite_below(F2 v) {
  float x, y;
  unpack(v, &x, &y);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-3.402823466e38f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(-3.402823466e38f));
  return pack(x, y);
}
// The activations in f32, on N packed pairs.  gelu_tanh is 0.5 x (1 + tanh u)
// = x / (1 + exp(-2u)) with u = sqrt(2/pi) (x + 0.044715 x^3): like SiLU and
// the sigmoid a quotient without cancellation.  Its relative error is 2^-21 and
// what the exponent's roundings make of its size in nats: 2 2^-24 of it for
// SiLU and the sigmoid (2^-17 at x = -87), 8 2^-24 for the tanh form, under
// the rounding of a 16-bit y.  The reciprocal is 0 where 1 + 2^z passes 2^126:
// results below |x| 2^-126 are 0.
template <int N>
__device__ __forceinline__ void activate_pairs(int act, F2 (&v)[N]) {
  if (act == kActNone) return;
  if (act == kActGeluTanh) {
    // exp(-2u) = 2^(x (c1 + c3 x^2))
    const F2 c1 = pack(-1.5957691216057308f * kLog2e), c3 = pack(-1.5957691216057308f * 0.044715f * kLog2e);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gate2(finite_below(v[j]), mul2(v[j], fma2(mul2(v[j], v[j]), c3, c1)));
  } else if (act == kActSilu) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gate2(finite_below(v[j]), mul2(v[j], pack(-kLog2e)));
  } else if (act == kActSigmoid) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gate2(pack(1.0f), mul2(v[j], pack(-kLog2e)));
  } else if (act == kActGelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = gelu2(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float x, y;
      unpack(v[j], &x, &y);
      v[j] = pack(relu(x), relu(y));
    }
  }
}
// Adds 2 N consecutive values from p + i on (16 bytes at a time).
template <int N>
__device__ __forceinline__ void add_vec(const void* p, long long i, int dtype, F2 (&v)[N]) {
  if (dtype == kF32) {
    const ulonglong2* s = reinterpret_cast<const ulonglong2*>(static_cast<const float*>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const ulonglong2 u = s[j];
      v[2 * j] = add2(v[2 * j], F2{u.x});
      v[2 * j + 1] = add2(v[2 * j + 1], F2{u.y});
    }
    return;
  }
  const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const uint4 u = s[j];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float lo, hi;
      unpack2(dtype, w[k], &lo, &hi);
      v[4 * j + k] = add2(v[4 * j + k], pack(lo, hi));
    }
  }
}
template <int N>
__device__ __forceinline__ void store_pairs(void* p, long long i, int dtype, const F2 (&v)[N]) {
  if (dtype == kF32) {
    ulonglong2* d = reinterpret_cast<ulonglong2*>(static_cast<float*>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) d[j] = make_ulonglong2(v[2 * j].v, v[2 * j + 1].v);
    return;
  }
  uint32_t w[N];
  if (dtype == kBf16) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float lo, hi;
      unpack(v[j], &lo, &hi);
      w[j] = pack2(kBf16, lo, hi);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float lo, hi;
      unpack(v[j], &lo, &hi);
      w[j] = pack2(kF16, lo, hi);
    }
  }
  uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i);
#pragma unroll
  for (int j = 0; j < N / 4; ++j) d[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

// Output (t, r) from its sum: the form for every size, stride and type.  Its
// many cases are long code: callers loop over it.
__device__ __forceinline__ void finish_one(const LinearArgs& a, int t, int r, float v) {
  if (a.bias != nullptr) v = __fadd_rn(v, load_f32(a.bias, r, a.bias_dtype));
  F2 p[1] = {pack(v, 0.0f)};
  activate_pairs<1>(a.act, p);
  float unused;
  unpack(p[0], &v, &unused);
  if (a.residual != nullptr)
    v = __fadd_rn(v, load_f32(a.residual, static_cast<long long>(t) * a.res_stride + r, a.res_dtype));
  store_f32(a.y, static_cast<long long>(t) * a.y_stride + r, a.out_dtype, v);
}
// 32 outputs of token t from row r on, where 16-byte accesses serve (a.vec,
// all 32 rows there).  `bias`: their bias in f32 in shared memory, or null.
__device__ __forceinline__ void finish_run(const LinearArgs& a, int t, int r, const float (&v)[32],
                                           const float* bias) {
  F2 p[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) p[j] = pack(v[2 * j], v[2 * j + 1]);
  if (bias != nullptr) add_vec<16>(bias, 0, kF32, p);
  activate_pairs<16>(a.act, p);
  if (a.residual != nullptr) add_vec<16>(a.residual, static_cast<long long>(t) * a.res_stride + r, a.res_dtype, p);
  store_pairs<16>(a.y, static_cast<long long>(t) * a.y_stride + r, a.out_dtype, p);
}
// finish_run for a whole warp's 32 tokens t0 + lane.  A lane's bytes lie a
// row's stride from its neighbour's, so they change hands in shared memory
// (`stage`, 2 KB; 16-byte chunks swapped by the row so that both sides are
// free of bank conflicts): a store then covers eight tokens' 64 bytes each
// instead of 16 bytes of 32 tokens, and a 16-bit residual comes in the same
// way.
constexpr int kRowBytes = 64;
template <bool F32>
__device__ __forceinline__ void finish_warp(const LinearArgs& a, int t0, int t_end, int r, const float (&v)[32],
                                            const float* bias, unsigned char* stage, int lane) {
  const auto chunk = [&](int row, int c) {
    return reinterpret_cast<uint4*>(stage + row * kRowBytes + ((c ^ ((row >> 1) & 3)) << 4));
  };
  const int row8 = lane >> 2, c4 = lane & 3;  // of a pass over eight tokens
  const bool moved = a.residual != nullptr && a.res_dtype != kF32;
  __syncwarp();
  if (moved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + 8 * i + row8;
      if (t < t_end)
        *chunk(8 * i + row8, c4) = *reinterpret_cast<const uint4*>(
            static_cast<const uint16_t*>(a.residual) + static_cast<long long>(t) * a.res_stride + r + 8 * c4);
    }
    __syncwarp();
  }
  F2 p[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) p[j] = pack(v[2 * j], v[2 * j + 1]);
  if (bias != nullptr) add_vec<16>(bias, 0, kF32, p);
  activate_pairs<16>(a.act, p);
  if (moved) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 u = *chunk(lane, c);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float lo, hi;
        unpack2(a.res_dtype, w[k], &lo, &hi);
        p[4 * c + k] = add2(p[4 * c + k], pack(lo, hi));
      }
    }
  } else if (a.residual != nullptr && t0 + lane < t_end) {
    add_vec<16>(a.residual, static_cast<long long>(t0 + lane) * a.res_stride + r, a.res_dtype, p);
  }
  if (F32) {  // 16 columns at a time
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h > 0) __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<ulonglong2*>(chunk(lane, c)) = make_ulonglong2(p[8 * h + 2 * c].v, p[8 * h + 2 * c + 1].v);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + 8 * i + row8;
        if (t < t_end)
          *reinterpret_cast<uint4*>(static_cast<float*>(a.y) + static_cast<long long>(t) * a.y_stride + r + 16 * h +
                                    4 * c4) = *chunk(8 * i + row8, c4);
      }
    }
    return;
  }
  uint32_t w[16];
  if (a.out_dtype == kBf16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float lo, hi;
      unpack(p[j], &lo, &hi);
      w[j] = pack2(kBf16, lo, hi);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float lo, hi;
      unpack(p[j], &lo, &hi);
      w[j] = pack2(kF16, lo, hi);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) *chunk(lane, c) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + 8 * i + row8;
    if (t < t_end)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.y) + static_cast<long long>(t) * a.y_stride + r + 8 * c4) =
          *chunk(8 * i + row8, c4);
  }
}
// Four outputs of token t from row r on (from shared memory's partial sums),
// `b` their bias.
__device__ __forceinline__ void finish_four(const LinearArgs& a, int t, int r, float4 v, const F2 (&b)[2]) {
  const int n = a.rows - r;
  if (n <= 0) return;
  F2 p[2] = {pack(v.x, v.y), pack(v.z, v.w)};
  if (a.bias != nullptr) {
    p[0] = add2(p[0], b[0]);
    p[1] = add2(p[1], b[1]);
  }
  activate_pairs<2>(a.act, p);
  float o[4];
  unpack(p[0], &o[0], &o[1]);
  unpack(p[1], &o[2], &o[3]);
  if (a.residual != nullptr) {
    const long long at = static_cast<long long>(t) * a.res_stride + r;
    if (a.res_dtype == kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) o[i] = __fadd_rn(o[i], static_cast<const float*>(a.residual)[at + i]);
    } else {
      uint16_t raw[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) raw[i] = static_cast<const uint16_t*>(a.residual)[at + i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = __fadd_rn(o[i], a.res_dtype == kBf16 ? bf16_to_f32(raw[i]) : __half2float(__ushort_as_half(raw[i])));
    }
  }
  const long long at = static_cast<long long>(t) * a.y_stride + r;
  if (a.vec && a.out_dtype != kF32 && n >= 4) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) =
        make_uint2(pack2(a.out_dtype, o[0], o[1]), pack2(a.out_dtype, o[2], o[3]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) store_f32(a.y, at + i, a.out_dtype, o[i]);
}
// A warp's 32 lanes by 32 columns of a tile from (p0, q0) on, through shared
// memory eight columns at a time, so that neighbouring lanes have
// neighbouring outputs whatever the sizes, strides and types.  swap: lanes
// are rows and columns tokens; p_end, q_end: where the tile's end.
constexpr int kStageFloats = 32 * 9;
__device__ __forceinline__ void finish_block(const LinearArgs& a, int p0, int q0, int p_end, int q_end,
                                             const float (&v)[32], float* stage, int lane) {
#pragma unroll 1
  for (int g = 0; g < 4 && q0 + 8 * g < q_end; ++g) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = g == 0 ? v[j] : g == 1 ? v[8 + j] : g == 2 ? v[16 + j] : v[24 + j];
      stage[a.swap ? 33 * j + lane : 9 * lane + j] = x;
    }
    __syncwarp();
    // The lane's row r of eight tokens t, t + step, ...
    const int r = a.swap ? p0 + lane : q0 + 8 * g + (lane & 7);
    const int t = a.swap ? q0 + 8 * g : p0 + (lane >> 3), step = a.swap ? 1 : 4;
    const int t_end = a.swap ? q_end : p_end;
    const int at = a.swap ? lane : 9 * (lane >> 3) + (lane & 7), apart = a.swap ? 33 : 36;
    if (r >= (a.swap ? p_end : q_end)) continue;
    const float b = a.bias != nullptr ? load_f32(a.bias, r, a.bias_dtype) : 0.0f;
    F2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = pack(stage[at + 2 * i * apart], stage[at + (2 * i + 1) * apart]);
    if (a.bias != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = add2(p[i], pack(b));
    }
    activate_pairs<4>(a.act, p);
    float o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack(p[i], &o[2 * i], &o[2 * i + 1]);
    if (a.residual != nullptr) {
      // The type is asked for once, so that the eight loads are under way
      // together.
      const long long from = static_cast<long long>(t) * a.res_stride + r, apart_by = a.res_stride * step;
      float v8[8] = {};
      if (a.res_dtype == kF32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (t + i * step < t_end) v8[i] = static_cast<const float*>(a.residual)[from + i * apart_by];
      } else {
        uint16_t raw[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (t + i * step < t_end) raw[i] = static_cast<const uint16_t*>(a.residual)[from + i * apart_by];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v8[i] = a.res_dtype == kBf16 ? bf16_to_f32(raw[i]) : __half2float(__ushort_as_half(raw[i]));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __fadd_rn(o[i], v8[i]);
    }
    const long long first = static_cast<long long>(t) * a.y_stride + r, on = a.y_stride * step;
    if (a.out_dtype == kF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t + i * step < t_end) static_cast<float*>(a.y)[first + i * on] = o[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t + i * step < t_end)
          static_cast<uint16_t*>(a.y)[first + i * on] =
              a.out_dtype == kBf16 ? f32_to_bf16(o[i]) : __half_as_ushort(__float2half_rn(o[i]));
    }
  }
}

// ---- operands that TMA cannot read ----------------------------------------------------

// Moves w down by `off` bytes (even, under 16): w[0..N - 4) are then whole.
template <int N>
__device__ __forceinline__ void realign(uint32_t (&w)[N], uint32_t off) {
  if (off & 8) {
#pragma unroll
    for (int i = 0; i < N - 2; ++i) w[i] = w[i + 2];
  }
  if (off & 4) {
#pragma unroll
    for (int i = 0; i < N - 3; ++i) w[i] = w[i + 1];
  }
  const uint32_t sh = (off & 2) * 8;
#pragma unroll
  for (int i = 0; i < N - 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], sh);
}
// The first n of eight elements, the others 0.
__device__ __forceinline__ uint4 first_of(uint4 v, int n) {
  uint32_t o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = n - 2 * i;  // elements of this word that exist
    if (left <= 0) o[i] = 0u;
    else if (left == 1) o[i] &= 0xffffu;
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// (volatile: stays behind the wait for the previous kernel, which may write it)
__device__ __forceinline__ uint4 ldg_word(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// The n (0..8) 16-bit elements at p, the others 0, from the one or two
// aligned 16-byte words that hold them (no other word is read).
__device__ __forceinline__ uint4 load_chunk(const uint16_t* p, int n) {
  if (n <= 0) return make_uint4(0, 0, 0, 0);
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
  const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) - off);
  const uint4 a = ldg_word(s);
  uint4 b = make_uint4(0, 0, 0, 0);
  if (off + 2 * n > 16) b = ldg_word(s + 1);
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  realign<8>(w, off);
  const uint4 v = make_uint4(w[0], w[1], w[2], w[3]);
  return n < 8 ? first_of(v, n) : v;
}

// ---- the tensor-core kernel -------------------------------------------------------------

struct __align__(128) LinearTail {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drained;
  uint32_t tmem_base;
  int abort;
  float bias[kEpiWarps][128];            // each epilogue warp's columns of a tile, in f32
};
// Behind the tail: each epilogue warp's memory for finish_block (kStageFloats)
// or, in the pair kernel, finish_warp.
constexpr int kPairStageBytes = 32 * kRowBytes;
static_assert(kPairStageBytes >= 4 * kStageFloats, "finish_block fits too");

// The bias of a warp's 32-column groups set, set + sets, ... (four at most) of
// the rows from r0 on, into its shared memory; null without a bias.
__device__ __forceinline__ const float* fetch_bias(const LinearArgs& a, float* mine, int r0, int set, int sets,
                                                   int lane) {
  if (a.bias == nullptr) return nullptr;
  __syncwarp();
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int r = r0 + 32 * (set + sets * g) + lane;
    mine[32 * g + lane] = r < a.rows ? load_f32(a.bias, r, a.bias_dtype) : 0.0f;
  }
  __syncwarp();
  return mine;
}

__device__ __forceinline__ void give_up(LinearTail* t) {
  atomicCAS(&g_status, 0, kErrTimeout);
  *reinterpret_cast<volatile int*>(&t->abort) = 1;
}
__device__ __forceinline__ bool gave_up(LinearTail* t) { return *reinterpret_cast<volatile int*>(&t->abort) != 0; }

struct Tile {
  int p0, q0;
};
// Tiles in groups of kGroup along P, so that those running together share
// rows of both operands in L2.
__device__ __forceinline__ Tile tile_of(const LinearArgs& a, int u, int height = kBM) {
  const int kGroup = 16 * kBM / height;
  const int per = kGroup * a.tiles_q;
  const int g = u / per, rest = u - g * per;
  const int size = min(kGroup, a.tiles_p - g * kGroup);
  Tile t;
  t.q0 = rest / size * a.bn;
  t.p0 = (g * kGroup + rest % size) * height;
  return t;
}

// CHUNKED: the accumulation is cut every `chunk` stages and carried on in
// registers (bn <= 128), for f32 outputs.
template <bool LOADERS, bool CHUNKED>
__global__ void __launch_bounds__(LOADERS ? kLoaderThreads : kMmaThreads, 1)
    k_linear_mma(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                 const __grid_constant__ LinearArgs a) {
  constexpr int kEpi = LOADERS ? kLoaderEpiWarps : kEpiWarps, kSets = kEpi / 4;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* ring = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const int slot = kABytes + a.bn * kBK * 2;
  LinearTail* tail = reinterpret_cast<LinearTail*>(ring + a.ring_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = a.stages;
  const int acc_cols = (a.bn + 31) & ~31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&tail->full[i], LOADERS ? kGroupWarps : 1);
      mbar_init(&tail->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tail->acc_full[i], 1);
      mbar_init(&tail->acc_empty[i], kEpi);
    }
    mbar_init(&tail->drained, 1);
    tail->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tail->tmem_base)),
                 "r"(a.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tail->tmem_base;
  pdl_wait();
  pdl_launch_dependents();

  // This CTA's share of the columns, and its tiles.
  const int rank = a.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int kb0 = static_cast<int>(static_cast<long long>(a.kblocks) * rank / a.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(a.kblocks) * (rank + 1) / a.splits);
  const int total = a.tiles_p * a.tiles_q;
  const int u0 = static_cast<int>(blockIdx.x) / a.splits;
  const int step = static_cast<int>(gridDim.x) / a.splits;
  const int chunk = CHUNKED ? a.chunk : kb1 - kb0;

  if (warp == 0) {
    if (!LOADERS) {
      // ---------------- producer ----------------
      int it = 0, st = 0;
      uint32_t phase = 1u;
      bool ok = true;
      for (int u = u0; ok && u < total; u += step) {
        const Tile w = tile_of(a, u);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          if (!__all_sync(kAll, mbar_wait_bounded(&tail->empty[st], phase, 1000ull * a.wait_us) && !gave_up(tail))) {
            give_up(tail);
            ok = false;
            break;
          }
          unsigned char* s = ring + st * slot;
          if (elect_one()) {
            mbar_arrive_expect_tx(&tail->full[st], static_cast<uint32_t>(slot));
            tma_load_2d(s, &map_p, kb * kBK, w.p0, &tail->full[st]);
            tma_load_2d(s + kABytes, &map_q, kb * kBK, w.q0, &tail->full[st]);
          }
          if (++st == stages) {
            st = 0;
            phase ^= 1u;
          }
        }
      }
      // Copies already issued land before the CTA can exit.
      for (int j = it > stages ? it - stages : 0; j < it; ++j)
        if (!mbar_wait_bounded(&tail->full[j % stages], (j / stages) & 1, 1000ull * a.wait_us)) give_up(tail);
    }
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    int st = 0, ai = 0;
    uint32_t phase = 0u;
    bool ok = true;
    const uint32_t idesc = idesc_f16(kBM, a.bn, a.dtype == kBf16);
    const uint64_t desc0 = sw128_desc(smem_u32(ring));
    for (int u = u0; ok && u < total; u += step) {
      for (int k = kb0; ok && k < kb1; k += chunk, ++ai) {
        const int buf = ai & 1;
        if (!__all_sync(kAll, !gave_up(tail) && mbar_wait_bounded(&tail->acc_empty[buf], ((ai >> 1) & 1) ^ 1u,
                                                                  1000ull * a.wait_us))) {
          give_up(tail);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + buf * acc_cols;
        const int end = min(kb1, k + chunk);
        for (int kb = k; kb < end; ++kb) {
          if (!__all_sync(kAll, mbar_wait_bounded(&tail->full[st], phase, 1000ull * a.wait_us))) {
            give_up(tail);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = desc0 + static_cast<uint32_t>(st * slot >> 4), db = da + (kABytes >> 4);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kBK / 16; ++i)
              umma_f16(d, da + 2 * i, db + 2 * i, idesc, (kb > k || i > 0) ? 1u : 0u);
            umma_commit(&tail->empty[st]);
          }
          __syncwarp();
          if (++st == stages) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (ok && elect_one()) umma_commit(&tail->acc_full[buf]);
        __syncwarp();
      }
    }
    // Every MMA issued has completed once `drained` flips.
    if (elect_one()) umma_commit(&tail->drained);
    __syncwarp();
    if (!mbar_wait_bounded(&tail->drained, 0, 1000ull * a.wait_us)) give_up(tail);
  } else if (warp < 2 + kEpi) {
    // ---------------- epilogue ----------------
    const int set = (warp - 2) >> 2;
    const int q = warp & 3;  // TMEM lane quarter this warp may read
    const int row = q * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q * 32) << 16);
    float* parts = reinterpret_cast<float*>(ring);  // [bn][128] of a split tile
    int ai = 0;
    for (int u = u0; u < total; u += step) {
      const Tile w = tile_of(a, u);
      const int valid = min(a.bn, a.q_rows - w.q0);
      const float* bias = nullptr;
      auto finish = [&](int c0, float(&v)[32]) {
        if (a.splits > 1) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c0 + j < valid) parts[(c0 + j) * kBM + row] = v[j];
        } else if (!a.swap && a.vec && c0 + 32 <= valid) {
          if (w.p0 + row < a.p_rows)
            finish_run(a, w.p0 + row, w.q0 + c0, v, bias != nullptr ? bias + c0 / (32 * kSets) * 32 : nullptr);
        } else {
          finish_block(a, w.p0 + 32 * q, w.q0 + c0, a.p_rows, w.q0 + valid, v,
                       reinterpret_cast<float*>(tail + 1) + (warp - 2) * kStageFloats, lane);
        }
      };
      if (!a.swap) bias = fetch_bias(a, tail->bias[warp - 2], w.q0, set, kSets, lane);
      if (!CHUNKED) {
        const int buf = ai & 1;
        const bool got = mbar_wait_bounded(&tail->acc_full[buf], (ai >> 1) & 1, 1000ull * a.wait_us);
        if (!__all_sync(kAll, got)) {
          if (lane == 0) give_up(tail);
          break;
        }
        tc_fence_after();
        for (int c0 = 32 * set; c0 < a.bn; c0 += 32 * kSets) {
          float v[32];
          tmem_ld32(lane_base + buf * acc_cols + c0, v);
          finish(c0, v);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->acc_empty[buf]);
        ++ai;
      } else {
        constexpr int kGroups = 2;  // 32-column groups of this warp
        float acc[kGroups][32];
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[g][j] = 0.0f;
        bool ok = true;
        for (int k = kb0; k < kb1; k += chunk, ++ai) {
          const int buf = ai & 1;
          const bool got = mbar_wait_bounded(&tail->acc_full[buf], (ai >> 1) & 1, 1000ull * a.wait_us);
          if (!__all_sync(kAll, got)) {
            if (lane == 0) give_up(tail);
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            const int c0 = 32 * (set + kSets * g);
            if (c0 < a.bn) {
#pragma unroll
              for (int h = 0; h < 32; h += 16) {
                float v[16];
                tmem_ld16(lane_base + buf * acc_cols + c0 + h, v);
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[g][h + j] = __fadd_rn(acc[g][h + j], v[j]);
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tail->acc_empty[buf]);
        }
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int c0 = 32 * (set + kSets * g);
          if (c0 < a.bn) finish(c0, acc[g]);
        }
      }
    }
  } else if (LOADERS) {
    // ---------------- loaders ----------------
    // Each warp serves up to kWarpRows consecutive rows of one side.  A row's
    // 64 columns lie in nine aligned 16-byte words at most; these come into the
    // warp's own buffers by cp.async (27 lanes, three rows a step), kAhead stages
    // ahead, and are then cut into the operand's 16-byte chunks (sixteen rows a
    // step).  A stage moves every row on by 128 bytes, so a row's offset in its
    // words stays the same over a tile.  Words without an element of the
    // operand are not read (size 0: zeros); rows beyond the operand are left
    // as they are, as nobody reads their products.
    const int group = (warp - (2 + kEpi)) / kGroupWarps, lw = (warp - (2 + kEpi)) % kGroupWarps;
    unsigned char* mine = ring + stages * slot + (warp - (2 + kEpi)) * (kAhead + 1) * kRawBytes;
    const int np = p_warps(a.bn);
    const bool side_p = lw < np;
    const int side_rows = side_p ? kBM : a.bn, side_warps = side_p ? np : kGroupWarps - np;
    const int each = (side_rows + side_warps - 1) / side_warps;
    const int r0 = (side_p ? lw : lw - np) * each;  // of the side's rows in a tile
    const int most = max(0, min(each, side_rows - r0));
    const int limit = side_p ? a.p_rows : a.q_rows;
    const long long pitch = (side_p ? a.p_stride : a.q_stride) * 2;
    // The rows that exist, and the first one's address.
    const auto rows_of = [&](int u, int* count) {
      const Tile w = tile_of(a, u);
      const int at = (side_p ? w.p0 : w.q0) + r0;
      *count = max(0, min(most, limit - at));
      return reinterpret_cast<uintptr_t>(side_p ? a.p : a.q) + (*count > 0 ? at * pitch : 0);
    };
    // The stage after the next one of the other group.
    const auto advance = [&](int* u, int* kb, int by) {
      for (int i = 0; i < by; ++i)
        if (++*kb == kb1) {
          *kb = kb0;
          *u += step;
        }
    };
    constexpr int kFetch = (kWarpRows + 2) / 3, kCut = kWarpRows / 16;
    const int half = lane & 1, row2 = lane >> 1;
    const int row3 = lane / 9, word = lane - 9 * row3;  // lanes 27 to 31 fetch nothing
    int iu = u0, ik = kb0, issued = 0, aimed = -1;
    advance(&iu, &ik, group);
    uintptr_t fetch_at = 0;
    int fetch_rows = 0;
    const auto issue = [&]() {
      if (iu < total) {
        if (iu != aimed) {
          fetch_at = rows_of(iu, &fetch_rows) + row3 * pitch;
          if (row3 == 3) fetch_rows = 0;
          aimed = iu;
        }
        const int bytes = 2 * min(kBK, a.cols - ik * kBK);
        const uintptr_t on = static_cast<uintptr_t>(ik) * (2 * kBK) + 16 * word;
        uint32_t to = smem_u32(mine) + issued % (kAhead + 1) * kRawBytes + row3 * 144 + 16 * word;
        uintptr_t at = fetch_at;
#pragma unroll
        for (int j = 0; j < kFetch; ++j) {
          if (row3 + 3 * j < fetch_rows) {
            const int off = static_cast<int>(at & 15u);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 432 * j), "l"(at - off + on),
                         "r"(16 * word < off + bytes ? 16 : 0)
                         : "memory");
          }
          at += 3 * pitch;
        }
        ++issued;
        advance(&iu, &ik, kLoadGroups);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int u = u0, kb = kb0, st = group, done = 0, cut = -1, cut_rows = 0;
    uint32_t phase = 1u, cut_at = 0u;  // cut_at: low bits of the address of the lane's first row
    const uint32_t pitch16 = 16u * static_cast<uint32_t>(pitch);
    advance(&u, &kb, group);
    for (int i = 0; i < kAhead; ++i) issue();
    while (u < total) {
      if (u != cut) {
        cut_at = static_cast<uint32_t>(rows_of(u, &cut_rows)) + static_cast<uint32_t>(row2) * static_cast<uint32_t>(pitch);
        cut = u;
      }
      issue();
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
      __syncwarp();
      if (!__all_sync(kAll, mbar_wait_bounded(&tail->empty[st], phase, 1000ull * a.wait_us) && !gave_up(tail))) {
        give_up(tail);
        break;
      }
      // The lane's half of rows r, r + 16: row r of P at slot, of Q at slot +
      // 16 KB, r * 128 either way, its chunks swapped by the row's low three
      // bits.  (Both sides are free of bank conflicts: four rows' halves per
      // 128 bytes.)
      const unsigned char* from = mine + done % (kAhead + 1) * kRawBytes + row2 * 144 + half * 64;
      unsigned char* to = ring + st * slot + (side_p ? 0 : kABytes) + (r0 + row2) * 128;
      const int count = a.cols - kb * kBK - 32 * half;
#pragma unroll
      for (int j = 0; j < kCut; ++j) {
        uint32_t w[20];
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          const uint4 v = reinterpret_cast<const uint4*>(from + 16 * 144 * j)[i];
          w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
        realign<20>(w, (cut_at + j * pitch16) & 15u);
        if (row2 + 16 * j < cut_rows) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 o = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            if (count < 32) o = first_of(o, count - 8 * i);
            *reinterpret_cast<uint4*>(to + 2048 * j + (((4 * half + i) ^ ((r0 + row2) & 7)) << 4)) = o;
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();  // (and the buffer has been read before it is filled again)
      if (lane == 0) mbar_arrive(&tail->full[st]);
      ++done;
      st += kLoadGroups;
      if (st >= stages) {
        st -= stages;
        phase ^= 1u;
      }
      advance(&u, &kb, kLoadGroups);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  if (a.splits > 1) {
    // Partial tiles lie in the CTAs' rings; CTA r adds up columns r,
    // r + splits, ... in rank order.  (Every thread comes here, whatever
    // happened before.)
    const Tile w = tile_of(a, u0);
    F2 bias[2] = {pack(0.0f), pack(0.0f)};  // of the lane's four rows, on its way during the barrier
    if (a.bias != nullptr) {
      float b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = w.p0 + 4 * lane + i;
        b[i] = r < a.rows ? load_f32(a.bias, r, a.bias_dtype) : 0.0f;
      }
      bias[0] = pack(b[0], b[1]);
      bias[1] = pack(b[2], b[3]);
    }
    __syncwarp();
    cluster_sync_all();
    if (!gave_up(tail)) {  // all warps: the roles are over
      const int valid = min(a.bn, a.q_rows - w.q0);
      const uint32_t parts = smem_u32(ring);
      for (int c = rank + warp * a.splits; c < valid; c += static_cast<int>(blockDim.x >> 5) * a.splits) {
        const uint32_t at = parts + (c * kBM + 4 * lane) * 4;
        float4 sum = ld_cluster_f4(at, 0);
        for (int r = 1; r < a.splits; ++r) {
          const float4 o = ld_cluster_f4(at, r);
          sum.x = __fadd_rn(sum.x, o.x);
          sum.y = __fadd_rn(sum.y, o.y);
          sum.z = __fadd_rn(sum.z, o.z);
          sum.w = __fadd_rn(sum.w, o.w);
        }
        finish_four(a, w.q0 + c, w.p0 + 4 * lane, sum, bias);
      }
    }
    __syncwarp();
    cluster_sync_all();  // the partial tiles stay until they have been read
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}

// ---- pairs of CTAs ----------------------------------------------------------------------
//
// k_linear_pair: two CTAs on one 256 x bn tile.  A stage brings 128 P rows and
// bn / 2 Q rows into each CTA, so a 256 x 256 tile loads 32 KB per CTA for 512
// cycles of MMA, where a CTA alone with 128 x 256 loads 48 KB: the traffic from
// L2 was what bound that one.  The even CTA issues the MMAs of both; full and
// acc_empty barriers are its own, commits arrive at empty and acc_full of both.
// CHUNKED: f32 outputs; a warp carries its 32 rows by 96 columns in registers
// (128 did not fit: 8192 x 8192 x 2048 271 us, with 96 242 us, on CTAs alone
// 329 us).
constexpr int kPairBn = 256, kPairChunkedBn = 192;

template <bool CHUNKED>
__global__ void __launch_bounds__(kMmaThreads, 1)
    k_linear_pair(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ LinearArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* ring = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const int slot = kABytes + a.bn / 2 * kBK * 2;
  LinearTail* tail = reinterpret_cast<LinearTail*>(ring + a.ring_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = a.stages;
  const uint32_t rank = cluster_rank();

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&tail->full[i], 1);
      mbar_init(&tail->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tail->acc_full[i], 1);
      mbar_init(&tail->acc_empty[i], 2 * kEpiWarps);
    }
    mbar_init(&tail->drained, 1);
    tail->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tail->tmem_base)),
                 "r"(a.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers and TMEM are there
  tc_fence_after();
  const uint32_t tmem = tail->tmem_base;
  pdl_wait();
  pdl_launch_dependents();
  const int total = a.tiles_p * a.tiles_q;
  const int u0 = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;

  if (warp == 0) {
    // ---------------- producer ----------------
    int it = 0, st = 0;
    uint32_t phase = 1u;
    bool ok = true;
    for (int u = u0; ok && u < total; u += step) {
      const Tile w = tile_of(a, u, 2 * kBM);
      const int p0 = w.p0 + static_cast<int>(rank) * kBM, q0 = w.q0 + static_cast<int>(rank) * (a.bn / 2);
      for (int kb = 0; kb < a.kblocks; ++kb, ++it) {
        if (!__all_sync(kAll, mbar_wait_bounded(&tail->empty[st], phase, 1000ull * a.wait_us) && !gave_up(tail))) {
          give_up(tail);
          ok = false;
          break;
        }
        unsigned char* s = ring + st * slot;
        const uint32_t bar = at_rank(&tail->full[st], 0);
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&tail->full[st], static_cast<uint32_t>(2 * slot));
          tma_load_2d_pair(s, &map_p, kb * kBK, p0, bar);
          tma_load_2d_pair(s + kABytes, &map_q, kb * kBK, q0, bar);
        }
        if (++st == stages) {
          st = 0;
          phase ^= 1u;
        }
      }
    }
    // Both CTAs' loads have landed once the even CTA's full barriers have
    // flipped.
    if (rank == 0)
      for (int j = it > stages ? it - stages : 0; j < it; ++j)
        if (!mbar_wait_bounded(&tail->full[j % stages], (j / stages) & 1, 1000ull * a.wait_us)) give_up(tail);
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------- MMA, for both CTAs ----------------
      int st = 0, ai = 0;
      uint32_t phase = 0u;
      bool ok = true;
      const uint32_t idesc = idesc_f16(2 * kBM, a.bn, a.dtype == kBf16);
      const uint64_t desc0 = sw128_desc(smem_u32(ring));
      const int chunk = CHUNKED ? a.chunk : a.kblocks;
      for (int at = 0, u = u0; ok && u < total; ++ai) {
        const int buf = ai & 1;
        if (!__all_sync(kAll, !gave_up(tail) && mbar_wait_bounded(&tail->acc_empty[buf], ((ai >> 1) & 1) ^ 1u,
                                                                  1000ull * a.wait_us))) {
          give_up(tail);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + buf * a.bn;
        const int end = min(a.kblocks, at + chunk);
        for (int kb = at; kb < end; ++kb) {
          if (!__all_sync(kAll, mbar_wait_bounded(&tail->full[st], phase, 1000ull * a.wait_us))) {
            give_up(tail);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = desc0 + static_cast<uint32_t>(st * slot >> 4), db = da + (kABytes >> 4);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kBK / 16; ++i)
              umma_f16_pair(d, da + 2 * i, db + 2 * i, idesc, (kb > at || i > 0) ? 1u : 0u);
            umma_commit_pair(&tail->empty[st]);
          }
          __syncwarp();
          if (++st == stages) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (ok && elect_one()) umma_commit_pair(&tail->acc_full[buf]);
        __syncwarp();
        at = end;
        if (at == a.kblocks) {
          at = 0;
          u += step;
        }
      }
      if (elect_one()) umma_commit_pair(&tail->drained);
      __syncwarp();
    }
  } else {
    // ---------------- epilogue ----------------
    const int set = (warp - 2) >> 2;
    const int q = warp & 3;
    unsigned char* stage = reinterpret_cast<unsigned char*>(tail + 1) + (warp - 2) * kPairStageBytes;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q * 32) << 16);
    int ai = 0;
    bool ok = true;
    for (int u = u0; ok && u < total; u += step) {
      const Tile w = tile_of(a, u, 2 * kBM);
      const int t0 = w.p0 + static_cast<int>(rank) * kBM + 32 * q;  // this warp's tokens
      const int valid = min(a.bn, a.q_rows - w.q0);
      const float* bias = fetch_bias(a, tail->bias[warp - 2], w.q0, set, 2, lane);
      const auto finish = [&](int c0, const float(&v)[32]) {
        if (a.vec && c0 + 32 <= valid)
          finish_warp<CHUNKED>(a, t0, a.p_rows, w.q0 + c0, v, bias != nullptr ? bias + c0 / 64 * 32 : nullptr, stage,
                               lane);
        else
          finish_block(a, t0, w.q0 + c0, a.p_rows, w.q0 + valid, v, reinterpret_cast<float*>(stage), lane);
      };
      const auto await = [&](int buf) {
        const bool got = mbar_wait_bounded(&tail->acc_full[buf], (ai >> 1) & 1, 1000ull * a.wait_us);
        if (!__all_sync(kAll, got)) {
          if (lane == 0) give_up(tail);
          return false;
        }
        tc_fence_after();
        return true;
      };
      const auto release = [&](int buf) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(at_rank(&tail->acc_empty[buf], 0));
      };
      if (!CHUNKED) {
        const int buf = ai & 1;
        if (!await(buf)) break;
        for (int c0 = 32 * set; c0 < a.bn; c0 += 64) {
          float v[32];
          tmem_ld32(lane_base + buf * a.bn + c0, v);
          finish(c0, v);
        }
        release(buf);
        ++ai;
      } else {
        constexpr int kGroups = kPairChunkedBn / 64;  // 32-column groups of this warp
        float acc[kGroups][32];
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[g][j] = 0.0f;
        for (int k = 0; k < a.kblocks; k += a.chunk, ++ai) {
          const int buf = ai & 1;
          if (!await(buf)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              float v[16];
              tmem_ld16(lane_base + buf * a.bn + 32 * set + 64 * g + h, v);
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[g][h + j] = __fadd_rn(acc[g][h + j], v[j]);
            }
          }
          release(buf);
        }
        if (!ok) break;
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = g == 0 ? acc[0][j] : g == 1 ? acc[1][j] : acc[2][j];
          if (32 * set + 64 * g < valid) finish(32 * set + 64 * g, v);
        }
      }
    }
  }
  // Every MMA has completed once `drained` flips, in either CTA.  The odd one,
  // which issues none, waits for it when its own tiles are done: a wait from
  // the start on would bound the whole product.
  __syncthreads();
  if (warp == 1 && !mbar_wait_bounded(&tail->drained, 0, 1000ull * a.wait_us)) give_up(tail);
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // neither CTA leaves while the other's MMAs, copies or arrivals may reach it
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}

// ---- one to four tokens -------------------------------------------------------------------

constexpr int kRowWarps = 8;
constexpr int kRowTokens = 4;

// acc[t] += sum of 8 products of a weight chunk with each token's chunk.
template <bool BF16, int NT>
__device__ __forceinline__ void dot8(const uint4 w, const uint4 (&x)[NT], float (&acc)[NT]) {
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float w0, w1;
    unpack2(BF16 ? kBf16 : kF16, ww[i], &w0, &w1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t xx = i == 0 ? x[t].x : i == 1 ? x[t].y : i == 2 ? x[t].z : x[t].w;
      float x0, x1;
      unpack2(BF16 ? kBf16 : kF16, xx, &x0, &x1);
      acc[t] = __fmaf_rn(w0, x0, acc[t]);
      acc[t] = __fmaf_rn(w1, x1, acc[t]);
    }
  }
}

// One weight row per group of `per_row` warps (1, 2, 4 or 8 of the CTA's 8);
// a lane takes the 8-column chunks lane, lane + 32 * per_row, ..., four in
// flight.  ALIGNED: every row of both operands starts on 16 bytes.
template <bool BF16, int NT, bool ALIGNED>
__global__ void __launch_bounds__(32 * kRowWarps) k_linear_rows(const __grid_constant__ LinearArgs a) {
  __shared__ float part[kRowWarps][NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_row = a.splits;
  const int r = (blockIdx.x * kRowWarps + warp) / per_row;
  const int sub = warp % per_row;
  pdl_wait();
  pdl_launch_dependents();
  float acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = 0.0f;
  if (r < a.rows) {
    const uint16_t* w = a.p + r * a.p_stride;
    const int chunks = (a.cols + 7) / 8, step = 32 * per_row;
    for (int c0 = sub * 32 + lane; c0 < chunks; c0 += 4 * step) {
      uint4 wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i * step, n = min(8, a.cols - 8 * c);
        if (ALIGNED && n == 8) wv[i] = ldg_stream(w + 8 * c);
        else wv[i] = load_chunk(w + (n > 0 ? 8 * c : 0), n);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i * step, n = min(8, a.cols - 8 * c);
        uint4 xv[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint16_t* x = a.q + t * a.q_stride;
          if (ALIGNED && n == 8) xv[t] = *reinterpret_cast<const uint4*>(x + 8 * c);
          else xv[t] = load_chunk(x + (n > 0 ? 8 * c : 0), n);
        }
        dot8<BF16, NT>(wv[i], xv, acc);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[t] = __fadd_rn(acc[t], __shfl_xor_sync(kAll, acc[t], o));
  }
  if (per_row > 1) {
    if (lane == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) part[warp][t] = acc[t];
    }
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      for (int s = 1; s < per_row; ++s) acc[t] = __fadd_rn(acc[t], part[warp + s][t]);
  }
  float mine = acc[0];  // lane t finishes token t
#pragma unroll
  for (int t = 1; t < NT; ++t) mine = lane == t ? acc[t] : mine;
  if (r < a.rows && lane < NT) finish_one(a, lane, r, mine);
}

// ---- host ------------------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [rows] rows of `cols` 16-bit elements, `stride` apart: boxes of 64 columns
// x box_rows rows, 128-byte swizzle, zeros outside.
bool operand_map(CUtensorMap* m, const void* base, int cols, int rows, long long stride, int box_rows, int dtype) {
  const auto fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t es[2] = {1, 1};
  return fn(m, dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
            const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tma_can_read(const void* base, int rows, long long stride) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && (rows == 1 || stride % 8 == 0) && stride < (1ll << 38);
}

template <auto Kern, typename... Args>
cudaError_t launch(int grid, int threads, size_t smem, int cluster, cudaStream_t st,
                   const Args&... args) {
  if (smem > 48 * 1024) {
    // Once per kernel and device, to the most that any plan asks for.
    static std::atomic<uint64_t> raised{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if ((raised.load(std::memory_order_relaxed) & bit) == 0) {
      e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
      if (e != cudaSuccess) return e;
      raised.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, Kern, args...);
}

template <bool BF16, int NT>
cudaError_t launch_rows(const LinearArgs& a, bool aligned, cudaStream_t st) {
  const int grid = static_cast<int>((static_cast<long long>(a.rows) * a.splits + kRowWarps - 1) / kRowWarps);
  return aligned ? launch<k_linear_rows<BF16, NT, true>>(grid, 32 * kRowWarps, 0, 1, st, a)
                 : launch<k_linear_rows<BF16, NT, false>>(grid, 32 * kRowWarps, 0, 1, st, a);
}
template <bool BF16>
cudaError_t launch_rows(const LinearArgs& a, bool aligned, cudaStream_t st) {
  switch (a.tokens) {
    case 1: return launch_rows<BF16, 1>(a, aligned, st);
    case 2: return launch_rows<BF16, 2>(a, aligned, st);
    case 3: return launch_rows<BF16, 3>(a, aligned, st);
    default: return launch_rows<BF16, 4>(a, aligned, st);
  }
}

// Clusters of each size that the current device runs at once with one CTA per
// SM (large ones do not fill it: its SMs come in groups of unequal size, and
// 15 clusters of 7 or 8 is what B200 has room for); asked once per device.
struct ClusterRoom {
  int clusters[9] = {};
};
cudaError_t cluster_room(int sms, ClusterRoom* out) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static ClusterRoom known[kDevices];  // clusters[1] is set last
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= kDevices) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  ClusterRoom& r = known[device];
  if (r.clusters[1] == 0) {
    constexpr int kSmem = 190 * 1024;
    const auto kern = k_linear_mma<false, false>;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
    if (e != cudaSuccess) return e;
    for (int size = 2; size <= 8; ++size) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(size);
      cfg.blockDim = dim3(kMmaThreads);
      cfg.dynamicSmemBytes = kSmem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = size;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if ((e = cudaOccupancyMaxActiveClusters(&r.clusters[size], kern, &cfg)) != cudaSuccess) return e;
    }
    r.clusters[1] = sms;
  }
  *out = r;
  return cudaSuccess;
}

// How a product is tiled.
struct Plan {
  double ns = 1e30;   // estimate, without the launch
  bool pair = false;  // k_linear_pair
  bool swap = false;  // w on the M side
  int bn = 64;        // N tile
  int splits = 1;     // CTAs that share a tile's columns
  int ring = 0;       // bytes of the operand ring
};

// The plan with the shortest estimate, over the tile widths, sides and splits
// that exist, and the pair kernel.  A CTA brings 130 bytes per ns into its shared memory (measured;
// loaders 29), a stage of the pair is bound by its MMAs (270 ns at bn = 256);
// partial tiles cost 1.2 us and more with their width, the last tile's
// epilogue in a CTA 0.6 us and 5 ns per column.  The ring is 96 KB, so
// that the next launch's CTAs can move in beside this one's; 200 KB was no
// faster but for the pair and for CTAs that run through many tiles.  f32
// outputs, which leave from registers, cost CTAs with several tiles 24 ns per
// column and tile more, and the pair 6 us per tile.
// The widths are what the sweeps ran.  w on the M side: tokens come in any
// number, and 96, 112 and 192 leave less of the last tile empty than the powers
// of two do (112 takes 333 tokens in three tiles).  x on the M side: rows are
// mostly multiples of 128, and a narrower tile only loads x more often.
// Measured against the best of a sweep (us, bf16 without an epilogue, the same
// operands again and again): 64 x 8192 x 2048 10.5 / 10.5, 128 x 2048 x 2048
// 8.1 / 8.1, 512 x 2048 x 2048 11.0 / 11.0.
Plan make_plan(const LinearArgs& a, bool tma, bool chunked, int sms, const ClusterRoom& room) {
  const int kblocks = (a.cols + kBK - 1) / kBK;
  const double rate = tma ? 130.0 : 29.0;
  Plan best;
  const auto consider = [&](bool swap, int bn, long long tiles, int splits) {
    const double waves = static_cast<double>((tiles * splits + sms - 1) / sms);
    const double stage = (kABytes + 128.0 * bn) / rate;
    double t = waves * ((kblocks + splits - 1) / splits) * stage + waves * 5.0 * bn + 600.0;
    if (chunked && splits == 1 && waves > 1) t += waves * 24.0 * bn;
    if (splits > 1) t += 1200.0 + 10.0 * bn;
    else if (swap) t += waves * 10.0 * bn;  // narrow stores
    if (t < best.ns) {
      best.ns = t;
      best.swap = swap;
      best.bn = bn;
      best.splits = splits;
      best.pair = false;
      best.ring = (waves > 2 ? 200 : 96) * 1024;
    }
  };
  const long long rows128 = (a.rows + kBM - 1) / kBM, tokens128 = (a.tokens + kBM - 1) / kBM;
  const int widest = !tma ? (chunked ? 64 : kLoadBn) : chunked ? 128 : 256;
  const int tokens16 = (a.tokens + 15) & ~15, rows16 = (a.rows + 15) & ~15;
  if (a.tokens <= 1024) {
    for (int bn : {16, 32, 64, 96, 112, 128, 192, 256}) {
      const int n = std::min(bn, tokens16);
      if (n > widest) break;
      const long long tiles = rows128 * ((a.tokens + n - 1) / n);
      consider(true, n, tiles, 1);
      // The most CTAs to a tile that run in one wave and have two blocks each.
      int s = std::min(8, kblocks / 2);
      while (s > 1 && tiles > room.clusters[s]) --s;
      if (s > 1) consider(true, n, tiles, s);
      if (n < bn) break;
    }
  }
  for (int bn : {64, 128, 256}) {
    const int n = std::min(bn, rows16);
    if (n > widest) break;
    consider(false, n, tokens128 * ((a.rows + n - 1) / n), 1);
    if (n < bn) break;
  }
  if (tma && a.tokens > 128 && a.rows > 128) {
    const int bn = chunked ? kPairChunkedBn : kPairBn;
    const long long tiles = static_cast<long long>((a.tokens + 255) / 256) * ((a.rows + bn - 1) / bn);
    const double waves = static_cast<double>((tiles + sms / 2 - 1) / (sms / 2));
    const double t = waves * (kblocks * 270.0 * bn / kPairBn + (chunked ? 6000.0 : 0.0)) + 600.0 + 5.0 * bn * 2;
    if (t < best.ns) {
      best.ns = t;
      best.pair = true;
      best.swap = false;
      best.bn = bn;
      best.splits = 1;
      best.ring = 200 * 1024;
    }
  }
  return best;
}

}  // namespace

static std::atomic<uint32_t> linear_wait_us{2000000u};
void set_linear_wait_limit(uint32_t us) { linear_wait_us.store(us, std::memory_order_relaxed); }

cudaError_t launch_linear_epilogue(LinearArgs a, const uint16_t* w, long long w_stride, const uint16_t* x,
                                   long long x_stride, cudaStream_t st) {
  DeviceAttrs dev;
  cudaError_t e = current_device_attrs(&dev);
  if (e != cudaSuccess) return e;
  a.wait_us = linear_wait_us.load(std::memory_order_relaxed);
  const auto aligned = [](const void* p, long long stride, int dtype) {
    const long long size = dtype == kF32 ? 4 : 2;
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0);
  };
  // (the bias is read an element at a time)
  a.vec = aligned(a.y, a.y_stride, a.out_dtype) && aligned(a.residual, a.res_stride, a.res_dtype);

  const bool tma = tma_can_read(w, a.rows, w_stride) && tma_can_read(x, a.tokens, x_stride);
  const bool chunked = a.out_dtype == kF32;
  const double row_ns = a.tokens > kRowTokens ? 1e30
                                              : 2600.0 + 500.0 * (a.tokens - 1) +
                                                    2.0 * a.rows * a.cols / 5500.0 * (0.7 + 0.3 * a.tokens);
  Plan plan;
  if (row_ns > 4000.0) {  // (no plan is faster than that)
    ClusterRoom room;
    if ((e = cluster_room(dev.sms, &room)) != cudaSuccess) return e;
    plan = make_plan(a, tma, chunked, dev.sms, room);
  }
  // One to four tokens on the CUDA cores, where that is faster: 2.6 us and
  // the weights at 5.5 TB/s, slower with every token more, against 4 us and
  // the plan (measured, one token: 512 x 2048 3.2 and 5.3 us, 2048 x 2048 3.8
  // and 5.9, 8192 x 2048 9.7 and 7.8; four: 5.5 and 5.4, 6.2 and 5.9, 15 and
  // 7.8).
  if (row_ns < 4000.0 + plan.ns) {
    a.p = w;
    a.p_stride = w_stride;
    a.q = x;
    a.q_stride = x_stride;
    // Warps per row: up to 8, while the GPU has fewer than 16 warps per SM
    // and a warp keeps a chunk per lane.
    int per = 1;
    while (per < kRowWarps && static_cast<long long>(a.rows) * per < 16ll * dev.sms && a.cols >= 512 * per) per *= 2;
    a.splits = per;
    const bool al = aligned(w, a.rows == 1 ? 0 : w_stride, kBf16) && aligned(x, a.tokens == 1 ? 0 : x_stride, kBf16);
    return a.dtype == kBf16 ? launch_rows<true>(a, al, st) : launch_rows<false>(a, al, st);
  }

  a.swap = plan.swap;
  const uint16_t* p = a.swap ? w : x;
  const uint16_t* q = a.swap ? x : w;
  a.p = p;
  a.q = q;
  a.p_rows = a.swap ? a.rows : a.tokens;
  a.q_rows = a.swap ? a.tokens : a.rows;
  a.p_stride = a.swap ? w_stride : x_stride;
  a.q_stride = a.swap ? x_stride : w_stride;
  a.bn = plan.bn;
  a.splits = plan.splits;
  const int height = plan.pair ? 2 * kBM : kBM;
  a.tiles_p = (a.p_rows + height - 1) / height;
  a.tiles_q = (a.q_rows + a.bn - 1) / a.bn;
  a.kblocks = (a.cols + kBK - 1) / kBK;
  a.chunk = kChunk;
  const int slot = kABytes + (plan.pair ? a.bn / 2 : a.bn) * kBK * 2;
  a.stages = tma ? std::min(kMaxStages, plan.ring / slot) : kLoadStages;
  a.ring_bytes = std::max(a.stages * slot + (tma ? 0 : kRawTotal), a.splits > 1 ? a.bn * kBM * 4 : 0);
  // Two accumulators, but one where a CTA has one tile and one accumulation.
  // CTAs of a cluster wait for one another while they hold TMEM: with at most
  // 256 of the 512 columns each, and shared memory for two per SM, no two
  // clusters on two streams can each hold what the other one needs.  (The
  // pair kernel takes all columns, and an SM to itself.)
  const bool single = a.splits > 1 && !chunked;
  int cols = 32;
  while (cols < (single ? 1 : 2) * ((a.bn + 31) & ~31)) cols *= 2;
  a.tmem_cols = cols;
  const size_t smem = 1024 + a.ring_bytes + sizeof(LinearTail) +
                      kEpiWarps * (plan.pair ? kPairStageBytes : sizeof(float) * kStageFloats);
  const long long tiles = static_cast<long long>(a.tiles_p) * a.tiles_q;

  CUtensorMap mp = {}, mq = {};
  if (tma) {
    const long long ps = a.p_rows == 1 ? (a.cols + 7) / 8 * 8 : a.p_stride;
    const long long qs = a.q_rows == 1 ? (a.cols + 7) / 8 * 8 : a.q_stride;
    if (!operand_map(&mp, p, a.cols, a.p_rows, ps, kBM, a.dtype) ||
        !operand_map(&mq, q, a.cols, a.q_rows, qs, plan.pair ? a.bn / 2 : a.bn, a.dtype))
      return cudaErrorInvalidValue;
  }
  if (plan.pair) {
    const int grid = 2 * static_cast<int>(std::min<long long>(tiles, dev.sms / 2));
    return chunked ? launch<k_linear_pair<true>>(grid, kMmaThreads, smem, 2, st, mp, mq, a)
                   : launch<k_linear_pair<false>>(grid, kMmaThreads, smem, 2, st, mp, mq, a);
  }
  const int grid = a.splits > 1 ? static_cast<int>(tiles) * a.splits
                                : static_cast<int>(std::min<long long>(tiles, dev.sms));
  if (tma)
    return chunked ? launch<k_linear_mma<false, true>>(grid, kMmaThreads, smem, a.splits, st, mp, mq, a)
                   : launch<k_linear_mma<false, false>>(grid, kMmaThreads, smem, a.splits, st, mp, mq, a);
  return chunked ? launch<k_linear_mma<true, true>>(grid, kLoaderThreads, smem, a.splits, st, mp, mq, a)
                 : launch<k_linear_mma<true, false>>(grid, kLoaderThreads, smem, a.splits, st, mp, mq, a);
}

cudaError_t take_linear_status(int* code, cudaStream_t st) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(code, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e != cudaSuccess || (e = cudaStreamSynchronize(st)) != cudaSuccess || *code == 0) return e;
  const int none = 0;
  if ((e = cudaMemcpyToSymbolAsync(g_status, &none, sizeof(int), 0, cudaMemcpyHostToDevice, st)) != cudaSuccess)
    return e;
  return cudaStreamSynchronize(st);
}

}  // namespace fw
