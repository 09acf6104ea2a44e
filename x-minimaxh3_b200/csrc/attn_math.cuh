// 16-bit element arithmetic shared by the attention kernels: bf16 or fp16
// storage, fp32 values, packed pairs in 32-bit words (low half first).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

#include <utility>

namespace h3 {

// Dependent launches: the kernels of one operator follow one another on a stream. The next
// one may start its CTAs once all of this one's have called launch_next(), and reads what
// this one writes only behind wait_previous(), which waits for its end. Every kernel of a
// chain waits before it writes anything, so nothing of it overlaps the kernel before.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// barrier of a cluster's CTAs in its two halves; stores before arrive are seen behind wait
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// kernel<<<grid, block, smem, stream>>>(args...) in clusters of `cluster` CTAs; after_previous:
// as a dependent of the launch before it
template <typename... P, typename... A>
cudaError_t launch_chained(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                           bool after_previous, int cluster, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  if (after_previous) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

constexpr int kHeadDim = 128;  // the head dim of every attention kernel of this library

template <bool F16>
struct Elem16 {
  static __device__ __forceinline__ float lo(uint32_t w) {
    if constexpr (F16) return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu)));
    return bf16_lo(w);
  }
  static __device__ __forceinline__ float hi(uint32_t w) {
    if constexpr (F16) return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
    return bf16_hi(w);
  }
  // two floats -> packed pair, each rounded to nearest even
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if constexpr (F16) {
      uint32_t r;
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
      return r;
    }
    return pack_bf16(lo, hi);
  }
  // c[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    if constexpr (F16)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Softmax weights are held as 2^BITS times exp(s - m) up to the end, where BITS cancels in O / l
// and is taken out of the log-sum-exp. fp16 has only 24 binary places below 1, so that weights
// below 2^-25 of the largest would be lost to P while l counts them: 32,760 keys at 2^-25.5
// are 0.07% of the row, more than fp16's own rounding of the result. BITS is what lies
// between the largest weight and 65,504. bf16 has fp32's range and needs none.
template <bool F16, int BITS>
struct WeightScale {
  static constexpr float log2 = F16 ? (float)BITS : 0.0f;
  static constexpr float inv = F16 ? 1.0f / (float)(1 << BITS) : 1.0f;
};

// two fp32 per instruction (sm_100 packed arithmetic, each half rounded to nearest)
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^a, 2^b by arithmetic on the FMA pipe, for a, b <= 64. n = round(x) through the addition
// of 1.5 * 2^23, f = x - n in [-0.5, 0.5], the polynomial of degree 5 with the least
// relative error there (Remez exchange; 2.4e-7 with these fp32 coefficients), times 2^n
// built from n's bits. 0 below -126.5, where n is -127 and those bits come out as 0 (the
// weight of a hidden key is exactly 0); NaN stays NaN.
__device__ __forceinline__ void exp2_poly2(uint64_t x, float& a, float& b) {
  float x0, x1;
  f2_unpack(x, x0, x1);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(x0), "f"(-127.0f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(x1), "f"(-127.0f));
  x = f2_pack(x0, x1);
  const uint64_t t = f2_add(x, f2_pack(12582912.0f, 12582912.0f));
  const uint64_t f = f2_fma(f2_add(t, f2_pack(-12582912.0f, -12582912.0f)), f2_pack(-1.0f, -1.0f), x);
  uint64_t y = f2_fma(f2_pack(0.0013276472454890609f, 0.0013276472454890609f), f,
                      f2_pack(0.009675540961325169f, 0.009675540961325169f));
  y = f2_fma(y, f, f2_pack(0.05550713092088699f, 0.05550713092088699f));
  y = f2_fma(y, f, f2_pack(0.24022120237350464f, 0.24022120237350464f));
  y = f2_fma(y, f, f2_pack(0.6931469440460205f, 0.6931469440460205f));
  y = f2_fma(y, f, f2_pack(1.0000001192092896f, 1.0000001192092896f));
  float t0, t1;
  f2_unpack(t, t0, t1);
  const uint32_t e0 = (__float_as_uint(t0) << 23) + 0x3F800000u, e1 = (__float_as_uint(t1) << 23) + 0x3F800000u;
  f2_unpack(f2_mul(y, f2_pack(__uint_as_float(e0), __uint_as_float(e1))), a, b);
}

// three-input maximum (sm_100); NaN operands are dropped, as by fmaxf
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// transpose of an 8 x 8 matrix of 16-bit values held one row per four lanes
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t w) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}

// 128-bit read-only load of data this SM reads once (no L1 line kept)
__device__ __forceinline__ uint4 ldg_stream_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

}  // namespace h3
