// The NVFP4 block recipe of the quantizers (quantize.cu, moe.cu): one block of 16 values -> its E4M3 scale
// byte and eight packed bytes, and the SiLU(gate) * up step in front of it.
#pragma once

#include "common.cuh"

namespace b2 {
namespace {

// SiLU(gate) * up on one packed pair, re-rounded to the input type
// (fp_quant.py silu_f32 :340-344, silu_and_mul_pair :363-372).
template <typename Tag>
__device__ __forceinline__ uint32_t silu_and_mul_pair(uint32_t gate, uint32_t up) {
  // The reference unpacks with a multiply by 1.0, which changes no bit of a finite value.
  const float2 s = mul_f32x2(silu_f32x2(unpack2<Tag>(gate)), unpack2<Tag>(up));
  return pack_from_f32<Tag>(s.x, s.y);
}

// The same for four pairs side by side: silu_f32x2 with one choice of path for all of them, so that their chains of
// dependent instructions overlap.
template <typename Tag>
__device__ __forceinline__ void silu_and_mul_4(const uint32_t (&gate)[4], const uint32_t (&up)[4], uint32_t (&out)[4]) {
  const float2 one = make_float2(1.0f, 1.0f), minus = make_float2(-1.0f, -1.0f);
  const float2 log2e = make_float2(-1.4426950408889634f, -1.4426950408889634f);
  constexpr float kTiny = 8.67361737988e-19f;  // 2^-60
  float2 g[4], e[4], s[4];
  bool fast = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    g[i] = unpack2<Tag>(gate[i]);
    const float2 t = mul_f32x2(g[i], log2e);
    e[i] = make_float2(ex2_approx_ftz(t.x), ex2_approx_ftz(t.y));
    fast = fast && fmaxf(fabsf(t.x), fabsf(t.y)) < 64.0f && fabsf(g[i].x) >= kTiny && fabsf(g[i].y) >= kTiny;
  }
  if (fast) {
    float2 nd[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = fma_f32x2(e[i], one, one);
      nd[i] = fma_f32x2(e[i], minus, minus);
      r[i] = make_float2(rcp_approx_ftz(d.x), rcp_approx_ftz(d.y));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fma_f32x2(r[i], fma_f32x2(nd[i], r[i], one), r[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = mul_f32x2(g[i], r[i]);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = fma_f32x2(fma_f32x2(nd[i], s[i], g[i]), r[i], s[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = fma_f32x2(e[i], one, one);
      s[i] = make_float2(__fdiv_rn(g[i].x, d.x), __fdiv_rn(g[i].y, d.y));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 m = mul_f32x2(s[i], unpack2<Tag>(up[i]));
    out[i] = pack_from_f32<Tag>(m.x, m.y);
  }
}

// One 16-element block held as 8 packed words -> (E4M3 scale byte, 64 packed E2M1 bits).
template <typename Tag>
__device__ __forceinline__ void quantize_block(const uint32_t (&w)[8], float gs, float rcp_gs,
                                               float rcp6, uint32_t& sf_byte, uint2& packed) {
  const uint32_t lo4[4] = {w[0], w[1], w[2], w[3]};
  const uint32_t hi4[4] = {w[4], w[5], w[6], w[7]};
  const uint32_t m2 = hmax2<Tag>(absmax_4<Tag>(lo4), absmax_4<Tag>(hi4));
  const float amax = pair_max_to_f32<Tag>(m2);
  // scale = gs * (amax * rcp(6)), two roundings, inner product first.
  const float scale = mul_f32(gs, mul_f32(amax, rcp6));
  sf_byte = cvt_f32_to_e4m3(scale) & 0xFFu;
  const float sf_f32 = e4m3_to_f32(sf_byte);
  // out_scale = rcp(sf * rcp(gs)), zero when the stored scale is zero.
  const float inv = rcp_approx_ftz(mul_f32(sf_f32, rcp_gs));
  const float out_scale = (sf_f32 == 0.0f) ? 0.0f : inv;
  // x * out_scale, two elements per mul.f32x2 (each half rounds like mul.f32)
  const float2 s2 = make_float2(out_scale, out_scale);
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = mul_f32x2(unpack2<Tag>(w[i]), s2);
    v[2 * i] = q.x;
    v[2 * i + 1] = q.y;
  }
  packed.x = cvt_e2m1x8(v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = mul_f32x2(unpack2<Tag>(w[4 + i]), s2);
    v[2 * i] = q.x;
    v[2 * i + 1] = q.y;
  }
  packed.y = cvt_e2m1x8(v);
}

template <bool V8>
__device__ __forceinline__ void load_block(const uint8_t* p, uint32_t (&w)[8]) {
  if constexpr (V8) {
    ld_stream_256(p, w);
  } else {
    uint32_t a[4], b[4];
    ld_stream_128(p, a);
    ld_stream_128(p + 16, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = a[i];
      w[4 + i] = b[i];
    }
  }
}

}  // namespace
}  // namespace b2
