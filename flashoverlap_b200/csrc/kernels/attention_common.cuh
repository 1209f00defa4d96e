// Device pieces that the attention kernels share: 16-bit conversions, asynchronous copies, warp matrix instructions.
#pragma once

#include <mutex>
#include <set>
#include <utility>

#include "attention.h"
#include "sm100_ptx.cuh"

namespace fo {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

template <bool BF16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t v;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
template <bool BF16>
__device__ __forceinline__ float widen(uint16_t u) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
  else return __half2float(__ushort_as_half(u));
}

// 2^x, 2^-inf = 0
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in a register pair, for the instructions that work on both.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair make_pair(float x, float y) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 split(Pair a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
// Larger of three, NaN if any is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x without the special function unit, which gives 16 results a clock and SM: x = n + f, |f| <= 1/2, a polynomial of degree 5
// that is exactly 1 at 0 (least squares of the relative error, reweighted until it was level: 1.7e-7 with its roundings in
// fp32), n added to the exponent.  x from -inf to 127; below -126.5 the result loses bits, from -127 down it is 0.  Not for
// NaN.
__device__ __forceinline__ float2 exp2_poly(Pair x) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to a whole number, which its low bits then hold
  const float2 u = split(x);
  x = make_pair(fmaxf(u.x, -127.f), fmaxf(u.y, -127.f));
  const Pair t = add2(x, make_pair(kRound, kRound));
  const Pair f = fma2(add2(t, make_pair(-kRound, -kRound)), make_pair(-1.f, -1.f), x);
  Pair r = make_pair(0.0013264727f, 0.0013264727f);
  r = fma2(r, f, make_pair(0.009671513f, 0.009671513f));
  r = fma2(r, f, make_pair(0.055507336f, 0.055507336f));
  r = fma2(r, f, make_pair(0.24022242f, 0.24022242f));
  r = fma2(r, f, make_pair(0.693147f, 0.693147f));
  r = fma2(r, f, make_pair(1.f, 1.f));
  const float2 n = split(t), y = split(r);
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)));
}

// 16 bytes to shared memory, past L1; zeros when `take` is false (the source is not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take) {
  const int n = take ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// An 8 x 8 matrix of 16-bit values, two of a row in each lane, the other way round.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// d[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums.
template <bool BF16>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Dynamic shared memory of a kernel, asked for once on each device.
template <typename... Params>
cudaError_t allow_smem(void (*kernel)(Params...), int bytes) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const std::pair<int, const void*> key(dev, reinterpret_cast<const void*>(kernel));
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(key)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.insert(key);
  return e;
}

// Launch whose CTAs may be placed while the kernel before it drains (they wait for it themselves).
template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                         int cluster, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace attn
}  // namespace fo
