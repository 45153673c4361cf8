// Shared device helpers for the NVFP4 hot path (sm_100a only).
//
// The quantizers must reproduce the reference's arithmetic bit for bit, so every
// floating-point step that matters is spelled as the exact PTX instruction the
// reference emits (tirx_kernels/flashinfer/utils/fp_quant.py): plain IEEE mul/add
// without .ftz and without fused contraction, MUFU approximations with .ftz, and
// the sm_100a-only e4m3x2 / e2m1x2 conversions.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200_nvfp4.h"

namespace b2 {

// ---- error plumbing (host) ---------------------------------------------------
void set_error(const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* what);

#define B2_CUDA_TRY(expr)                                  \
  do {                                                     \
    cudaError_t _e = (expr);                               \
    if (_e != cudaSuccess) return ::b2::cuda_fail(_e, #expr); \
  } while (0)

int device_sm_count();

struct F16Tag {};
struct BF16Tag {};

// ---- scalar arithmetic, pinned to the reference's instruction choice -----------
__device__ __forceinline__ float mul_f32(float a, float b) { return __fmul_rn(a, b); }  // mul.f32
__device__ __forceinline__ float add_f32(float a, float b) { return __fadd_rn(a, b); }  // add.f32

__device__ __forceinline__ float rcp_approx_ftz(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float rsqrt_approx_ftz(float a) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float lg2_approx(float a) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float ex2_approx(float a) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float ex2_approx_ftz(float a) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float max_f32(float a, float b) {
  float r;
  asm("max.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_f32(float a, float b) {
  float r;
  asm("min.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two independent IEEE multiplies in one instruction (mul.f32x2, sm_100): each half is rounded
// exactly like mul.f32, so results are bit-identical to the scalar form at half the issue cost.
__device__ __forceinline__ float2 mul_f32x2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 ra, rb, rd; mov.b64 ra, {%2, %3}; mov.b64 rb, {%4, %5}; mul.f32x2 rd, ra, rb;"
      " mov.b64 {%0, %1}, rd; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// Two independent fused multiply-adds (fma.rn.f32x2, sm_100); each half rounds exactly like fma.rn.f32.
__device__ __forceinline__ float2 fma_f32x2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{ .reg .b64 ra, rb, rc, rd; mov.b64 ra, {%2, %3}; mov.b64 rb, {%4, %5}; mov.b64 rc, {%6, %7};"
      " fma.rn.f32x2 rd, ra, rb, rc; mov.b64 {%0, %1}, rd; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// SiLU of two fp32 values, g / (1 + 2^(-g * log2 e)) with the quotient correctly rounded, bit for bit
// what mul.f32 + ex2.approx.ftz.f32 + add.f32 + div.rn.f32 give per element.  The common case runs
// the division as a Newton-refined reciprocal and two remainder corrections on packed FMAs (seven
// fma.rn.f32x2 for the pair); every remainder is exact there, so the last FMA rounds the true
// quotient.  Inputs outside that case (|g| >= 44: the denominator leaves the range where the
// reciprocal is normal; |g| < 2^-60, zero included: remainders underflow and a signed zero would be
// lost; NaN) take div.rn.f32.  EXACT_ONLY forces div.rn.f32 everywhere (the probe compares the two).
template <bool EXACT_ONLY = false>
__device__ __forceinline__ float2 silu_f32x2(float2 g) {
  const float2 t = mul_f32x2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 e = make_float2(ex2_approx_ftz(t.x), ex2_approx_ftz(t.y));
  const float2 one = make_float2(1.0f, 1.0f);
  const float2 d = fma_f32x2(e, one, one);  // e + 1, one rounding: add.f32
  constexpr float kTiny = 8.67361737988e-19f;  // 2^-60
  const bool fast = !EXACT_ONLY && fabsf(t.x) < 64.0f && fabsf(t.y) < 64.0f && fabsf(g.x) >= kTiny &&
                    fabsf(g.y) >= kTiny;  // every comparison is false for a NaN
  if (fast) {
    const float2 minus = make_float2(-1.0f, -1.0f);
    const float2 nd = fma_f32x2(e, minus, minus);  // -(e + 1), the same rounding
    float2 r = make_float2(rcp_approx_ftz(d.x), rcp_approx_ftz(d.y));
    r = fma_f32x2(r, fma_f32x2(nd, r, one), r);
    float2 q = mul_f32x2(g, r);
    q = fma_f32x2(fma_f32x2(nd, q, g), r, q);
    q = fma_f32x2(fma_f32x2(nd, q, g), r, q);
    return q;
  }
  return make_float2(__fdiv_rn(g.x, d.x), __fdiv_rn(g.y, d.y));
}

// ---- packed 16-bit pairs ---------------------------------------------------------
__device__ __forceinline__ uint32_t habs2(uint32_t x) { return x & 0x7FFF7FFFu; }

template <typename Tag>
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t hmax2<F16Tag>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t hmax2<BF16Tag>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename Tag>
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t hmul2<F16Tag>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t hmul2<BF16Tag>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename Tag>
__device__ __forceinline__ float unpack_lo(uint32_t w);
template <typename Tag>
__device__ __forceinline__ float unpack_hi(uint32_t w);
template <>
__device__ __forceinline__ float unpack_lo<BF16Tag>(uint32_t w) {
  return __uint_as_float(w << 16);
}
template <>
__device__ __forceinline__ float unpack_hi<BF16Tag>(uint32_t w) {
  return __uint_as_float(w & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ float unpack_lo<F16Tag>(uint32_t w) {
  float r;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, lo; }" : "=f"(r) : "r"(w));
  return r;
}
template <>
__device__ __forceinline__ float unpack_hi<F16Tag>(uint32_t w) {
  float r;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, hi; }" : "=f"(r) : "r"(w));
  return r;
}

template <typename Tag>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  return make_float2(unpack_lo<Tag>(w), unpack_hi<Tag>(w));
}

// cvt.rn.{f16,bf16}.f32 on two scalars, packed {lo, hi}.
template <typename Tag>
__device__ __forceinline__ uint32_t pack_from_f32(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_from_f32<F16Tag>(float lo, float hi) {
  uint32_t r;
  asm("{ .reg .b16 a, b; cvt.rn.f16.f32 a, %1; cvt.rn.f16.f32 b, %2; mov.b32 %0, {a, b}; }"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack_from_f32<BF16Tag>(float lo, float hi) {
  uint32_t r;
  asm("{ .reg .b16 a, b; cvt.rn.bf16.f32 a, %1; cvt.rn.bf16.f32 b, %2; mov.b32 %0, {a, b}; }"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
}

// Two values to 16 bits in one instruction.
template <typename Tag>
__device__ __forceinline__ uint32_t pack_pair(float2 v);
template <>
__device__ __forceinline__ uint32_t pack_pair<F16Tag>(float2 v) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack_pair<BF16Tag>(float2 v) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(v.y), "f"(v.x));
  return r;
}

// Tree abs-max over four packed words (8 values), then the max of the two lanes as fp32.
template <typename Tag>
__device__ __forceinline__ uint32_t absmax_4(const uint32_t (&v)[4]) {
  return hmax2<Tag>(hmax2<Tag>(habs2(v[0]), habs2(v[1])), hmax2<Tag>(habs2(v[2]), habs2(v[3])));
}
template <typename Tag>
__device__ __forceinline__ float pair_max_to_f32(uint32_t w) {
  return max_f32(unpack_lo<Tag>(w), unpack_hi<Tag>(w));
}

// ---- FP8 / FP4 conversions -----------------------------------------------------------
// cvt.rn.satfinite.e4m3x2.f32 {0, a}: the E4M3 byte of `a` (round to nearest even, saturating).
__device__ __forceinline__ uint32_t cvt_f32_to_e4m3(float a) {
  uint16_t p;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(0.0f), "f"(a));
  return static_cast<uint32_t>(p);
}
// Exact decode of an E4M3 byte through cvt.rn.f16x2.e4m3x2.
__device__ __forceinline__ float e4m3_to_f32(uint32_t code) {
  float r;
  asm("{ .reg .b16 lo, hi; .reg .b32 h2; cvt.rn.f16x2.e4m3x2 h2, %1; mov.b32 {lo, hi}, h2;"
      " cvt.f32.f16 %0, lo; }"
      : "=f"(r)
      : "h"(static_cast<uint16_t>(code)));
  return r;
}
// Eight fp32 values (element order) -> 8 E2M1 nibbles, element 0 in the lowest nibble.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{ .reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3}; }"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// ---- scale-factor layouts -------------------------------------------------------------
__device__ __host__ __forceinline__ int64_t sf_offset_128x4(int row, int col, int padded_cols) {
  return (int64_t)(col & 3) + (int64_t)(col >> 2) * 512 + (int64_t)(row & 31) * 16 +
         (int64_t)((row & 127) >> 5) * 4 + (int64_t)(row >> 7) * (128 * (int64_t)padded_cols);
}
__device__ __host__ __forceinline__ int64_t sf_offset_8x4(int row, int col, int padded_cols) {
  const int num_k_tiles = (padded_cols + 3) / 4;
  return (int64_t)(row >> 3) * ((int64_t)num_k_tiles * 32) + (int64_t)(col >> 2) * 32 +
         (int64_t)(row & 7) * 4 + (int64_t)(col & 3);
}

// ---- memory ---------------------------------------------------------------------------
// One 256-bit streaming load (read once, never reused).
__device__ __forceinline__ void ld_stream_256(const void* p, uint32_t (&r)[8]) {
  asm volatile(
      "ld.global.nc.L1::no_allocate.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "l"(p));
}
__device__ __forceinline__ void ld_stream_128(const void* p, uint32_t (&r)[4]) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "l"(p));
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace b2
