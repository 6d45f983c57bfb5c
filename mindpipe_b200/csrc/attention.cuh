// What the attention kernels share: the two 16-bit types, warp-level matrix products on tiles in shared memory, and the
// views of strided rows and of the paged cache.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "tc.cuh"

namespace mp {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -INFINITY;

// bits of the word that a call's kernels set where an index they were given is out of range
constexpr int kBadIndex = 1;

__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ uint32_t bits(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }

// Two fp32 values rounded to a pair of the type; a pair widened.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return bits(__floats2half2_rn(a, b)); }
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return bits(__floats2bfloat162_rn(a, b)); }
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }

// d[16 x 8] += a[16 x 16] b[16 x 8]
template <typename T> __device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// 16 bytes global -> shared, past L1; with `valid` false nothing is read and the 16 bytes become zero.
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace attn

// A [rows, heads, D] operand with strides in values; the last dimension is dense.
struct HeadRows {
  const char* data;
  long long token_stride, head_stride;      // bytes
};

// keys or values of the cache, [pages, heads, page size, D] with strides in bytes
struct CacheSide {
  char* data;
  long long page_stride, head_stride, token_stride;
};

// x / d and x % d for 0 <= x < 2^31 with a multiplication (d >= 1)
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv make_fast_div(uint32_t d) {
  uint32_t shift = 0;
  while ((1ull << shift) < d) ++shift;
  // mul = ceil(2^(32 + shift) / d) - 2^32: x / d = (hi(x mul) + x) >> shift; the sum is below 2^32 for x < 2^31
  const uint64_t mul = ((1ull << 32) * ((1ull << shift) - d)) / d + 1;
  return FastDiv{d, static_cast<uint32_t>(mul), shift};
}
__device__ __forceinline__ int fast_div(int x, const FastDiv& f) {
  return static_cast<int>((__umulhi(static_cast<uint32_t>(x), f.mul) + static_cast<uint32_t>(x)) >> f.shift);
}

// Checks that the entries share (host): a status.
int check_head_rows(const mp_head_rows* r, int D, HeadRows* out);
int check_cache(const mp_paged_cache* c, int D, CacheSide* k, CacheSide* v);

}  // namespace mp
