// Shared by the kernels around the paged 4-bit KV cache.
#pragma once

#include "common.cuh"

namespace uniql {

constexpr int kMaxTokens = 1 << 28;   // lengths and counts of tokens, pages and table columns: sums of two fit an int

// log2 of a supported page size, or -1
static inline int page_shift_of(int64_t page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (int64_t)1 << s) return s;
  return -1;
}

// Shape of a cache and of the heads it holds.
static inline int kv4_check(int64_t num_pages, int64_t page_size, int64_t dp, int64_t kv_heads, int64_t dk, int64_t dv) {
  if (page_shift_of(page_size) < 0 || (dp != 64 && dp != 128)) return UNIQL_ESHAPE;
  if (dk % 8 || dv % 8 || dk > dp || dv > dp) return UNIQL_ESHAPE;
  if (num_pages > kMaxTokens || kv_heads > 1024) return UNIQL_ESHAPE;
  return UNIQL_OK;
}

template <typename P>
static int launch_pdl(void (*kernel)(const P), unsigned ctas, int threads, size_t smem, cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  UNIQL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return UNIQL_OK;
}

// Quotient by a divisor that the host knows (Granlund and Montgomery: division by invariant integers), for n below 2^31.
struct FastDiv {
  uint32_t d, mul, shift;
  explicit FastDiv(uint32_t div = 1) : d(div), mul(0), shift(0) {
    while (((uint64_t)1 << shift) < div) ++shift;               // 2^shift >= div
    mul = (uint32_t)((((uint64_t)1 << (31 + shift)) + div - 1) / div);   // at most 2^32 - 1 for div > 1: see quot
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const {
    return d == 1 ? n : (uint32_t)(((uint64_t)n * mul) >> 31) >> shift;
  }
};

// Two floats side by side: one instruction of the FMA pipe for both (sm_100).
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The two nibbles at bits [3:0] and [19:16] of w as exact fp16 (c - bias), bias given as the fp16 pair 1024 + bias; and those at
// bits [7:4] and [23:20], where 1024 + 16 c is brought down with one fused multiply-add.
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, uint32_t sub) {
  const uint32_t t = lop3_and_or(w, 0x000f000fu, 0x64006400u);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&sub));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t kv4_pair_hi(uint32_t w, uint32_t add) {
  const uint32_t t = lop3_and_or(w, 0x00f000f0u, 0x64006400u);
  const uint32_t mul = 0x2c002c00u;             // 1/16
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&mul),
                            *reinterpret_cast<const __half2*>(&add));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// c[e] = codes (e, e + 4) of a word as fp16
__device__ __forceinline__ void kv4_codes(uint32_t w, uint32_t (&c)[4]) {
  const uint32_t w8 = w >> 8;
  c[0] = kv4_pair(w, 0x64006400u);
  c[1] = kv4_pair_hi(w, 0xd400d400u);           // -64
  c[2] = kv4_pair(w8, 0x64006400u);
  c[3] = kv4_pair_hi(w8, 0xd400d400u);
}

}  // namespace uniql
