// kv8_attn.cuh — what the attention kernels over the 8-bit cache share
// (kv8_attn.cu: few query rows; kv8_prompt.cu: prompts): their arguments, the
// f16 MMA and the conversion of codes to f16.
#pragma once

#include "kernels.cuh"
#include "ops.cuh"

namespace wg {

constexpr float KV8_LOG2E = 1.4426950408889634f;

struct Kv8AttnArgs {
  const int8_t* codes;
  const float* scales;
  int num_pages, shift, H, G;
  const void* q;
  int64_t ldq;
  int qdt;
  const int* cu_q;
  int n_q;
  const int* kv_lens;
  const int* table;
  int64_t ldt;
  int max_pages, R;
  int tiles, splits, causal, max_q;  // tiles: of kv8_prompt.cu
  float scale;
  void* out;
  int64_t ldo;
  int odt;
  bool q_vec, o_vec;  // rows that start on 16 bytes
};


constexpr int KV8_MAX_ATTN_ROWS = 1 << 30;  // (query, grouped head) rows of one request and K/V head
constexpr int KV8_MAX_SPLIT = 16;  // CTAs that share the tokens of a tile, or of a few rows (a cluster)

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a * b
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma16816_zero(d, a[0], a[1], a[2], a[3], b0, b1);
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  const uint32_t a[4] = {a0, a1, a2, a3};
  mma16816(c, a, b0, b1);
}
// Transposes an 8 x 8 matrix of 16-bit values held as row g, columns 2t and 2t + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Two bytes of w (already offset by 128: code + 128) as an f16 pair of codes:
// 0x6400 | u is 1024 + u, exact, and so is its difference from 1152.
template <int SEL>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
  const uint32_t h = __byte_perm(w, 0x64646464u, SEL);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Powers of two that take a row of bf16 or fp32 queries into f16 and back, from
// its largest magnitude: that goes to [2^14, 2^15), so bf16 values stay exact
// down to 2^-31 of it and fp32 values keep 11 bits down to 2^-28 of it (as long
// as it is 2^-112 or more).
__device__ __forceinline__ void query_range(float largest, float* up, float* down) {
  const int k = max((int)(__float_as_uint(largest) >> 23) - 127, -112);
  *up = __uint_as_float((uint32_t)(127 + 14 - k) << 23);
  *down = __uint_as_float((uint32_t)(127 - 14 + k) << 23);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
// A pair of softmax weights, at most 2^KV8_LIFT for the row's largest, as f16.
// Lifted, a weight is rounded by at most 2^-11 of itself down to 2^-28 of the
// largest, and by at most 2^-39 of the largest below that; unlifted, weights
// under 2^-25 would vanish, which under one strong token costs 60000 weak ones
// 1e-3 of the row's mass. An exponent above the lift (the rounding of scores of
// 2^25 and more) saturates.
constexpr float KV8_LIFT = 14.f;
constexpr float KV8_UNLIFT = 1.f / 16384.f;
__device__ __forceinline__ uint32_t pack_weights(float a, float b) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// 2^x, x <= KV8_LIFT (hardware approximation, 2^-22 relative; 0 for -inf)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// Launches of the prompt kernel (kv8_prompt.cu); tiles and splits are set here.
int launch_kv8_prompt(Kv8AttnArgs a, int head_dim, int64_t max_kv, cudaStream_t st);
int kv8_prompt_attributes();

}  // namespace wg
