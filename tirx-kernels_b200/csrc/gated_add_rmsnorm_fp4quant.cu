// The residual stream between two blocks of a transformer, one pass over its rows, for sm_100a:
//
//   u = x * rsqrt(mean(x^2) + eps) * w_post        the norm after the block (u = x without w_post)
//   h = c * residual + gate * u                    gate: one row per `rows_per_gate` rows (1 without gate)
//   y = h16 * rsqrt(mean(h16^2) + eps) * w_pre     the norm before the next block; h16 is h as it is stored
//
// h16 is written as the new residual, y in the 16-bit type or quantized to NVFP4 (one E4M3 scale per 16 values,
// gs * max|y| / 6 rounded to nearest, row-major or in 128 x 4 tiles; values y * gs / scale rounded to nearest E2M1).  Sums of squares, norms and
// h are fp32; h is rounded once, to the type it is stored in, and the second norm uses the rounded value so that it is
// the norm of what the next block's residual will read.  The product of a 16-bit value and a 16-bit weight is exact in
// fp32, so it is taken first and every value sees one or two roundings in front of its last one.
//
// The row stays in registers between the two reductions: x and the residual are read once, h and y written once,
// which is the floor.  A thread has units of 16 values, one 256-bit access each and, quantized, one scale block.
#include <algorithm>

#include "norm_quant.cuh"

namespace b2 {
namespace {

struct GatedParams {
  const uint8_t* x;
  const uint8_t* residual;
  const uint8_t* w_post;  // [H] or null
  const uint8_t* gate;    // [ceil(M / rows_per_gate), H] or null
  const uint8_t* w_pre;   // [H]
  uint8_t* residual_out;  // may be `residual`
  uint8_t* y;             // [M, H] in the input type, or uint8 [M, H / 2]
  uint8_t* sf;
  const float* gs;
  int M, H, units;        // units = H / 16
  int rows_per_gate;
  int sf_pad_cols;        // > 0: 128 x 4 tiles
  float scale, eps;
};

__device__ __forceinline__ void ld_256(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
__device__ __forceinline__ void ld_weight_256(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
__device__ __forceinline__ void st_256(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Sum over the threads of a row; `red` has a slot per warp of this row.
__device__ __forceinline__ float row_sum(float v, float* red, int warps, int warp, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (warps == 1) return v;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < warps ? red[lane] : 0.0f;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// 1 / sqrt(mean + eps), correctly rounded steps: once per row, and the quantizer's borders see every unit in the last place.
__device__ __forceinline__ float inverse_root(float sum, const GatedParams& p) {
  return __frcp_rn(__fsqrt_rn(__fdiv_rn(sum, static_cast<float>(p.H)) + p.eps));
}

// blockDim = (threads per row, rows per CTA); more than one row per CTA only with 32 threads per row.  V units per thread.
template <typename Tag, int V, bool QUANT>
__global__ void __launch_bounds__(1024) gated_add_rmsnorm_kernel(const __grid_constant__ GatedParams p) {
  __shared__ float red[2][32];
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
  pdl_wait();
  pdl_launch_dependents();
  if (row >= p.M) return;  // whole warps, and only where no warp waits for another
  const int64_t at = static_cast<int64_t>(row) * p.H * 2;
  uint32_t x[V][8], h[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int u = t + j * blockDim.x;
    if (u < p.units) {
      ld_256(p.x + at + static_cast<int64_t>(u) * 32, x[j]);
      ld_256(p.residual + at + static_cast<int64_t>(u) * 32, h[j]);
    }
  }
  float rstd = 1.0f;
  if (p.w_post) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (t + j * static_cast<int>(blockDim.x) < p.units) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = unpack2<Tag>(x[j][i]);
          sum = fmaf(f.x, f.x, sum);
          sum = fmaf(f.y, f.y, sum);
        }
      }
    }
    rstd = inverse_root(row_sum(sum, red[0], warps, warp, lane), p);
  }
  const uint8_t* gate = p.gate ? p.gate + static_cast<int64_t>(row / p.rows_per_gate) * p.H * 2 : nullptr;
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int u = t + j * blockDim.x;
    if (u < p.units) {
      uint32_t w[8], g[8];
      if (p.w_post) ld_weight_256(p.w_post + static_cast<int64_t>(u) * 32, w);
      if (gate) ld_weight_256(gate + static_cast<int64_t>(u) * 32, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float2 v = unpack2<Tag>(x[j][i]);
        if (p.w_post) {
          const float2 f = unpack2<Tag>(w[i]);
          v = make_float2(v.x * f.x * rstd, v.y * f.y * rstd);
        }
        if (gate) {
          const float2 f = unpack2<Tag>(g[i]);
          v = make_float2(v.x * f.x, v.y * f.y);
        }
        const float2 r = unpack2<Tag>(h[j][i]);
        h[j][i] = pack_from_f32<Tag>(fmaf(p.scale, r.x, v.x), fmaf(p.scale, r.y, v.y));
        const float2 s = unpack2<Tag>(h[j][i]);
        sum = fmaf(s.x, s.x, sum);
        sum = fmaf(s.y, s.y, sum);
      }
      st_256(p.residual_out + at + static_cast<int64_t>(u) * 32, h[j]);
    }
  }
  rstd = inverse_root(row_sum(sum, red[1], warps, warp, lane), p);
  const float gs = QUANT ? __ldg(p.gs) : 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int u = t + j * blockDim.x;
    if (u < p.units) {
      uint32_t w[8];
      ld_weight_256(p.w_pre + static_cast<int64_t>(u) * 32, w);
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = unpack2<Tag>(h[j][i]), g = unpack2<Tag>(w[i]);
        v[2 * i] = f.x * g.x;
        v[2 * i + 1] = f.y * g.y;
      }
      if constexpr (!QUANT) {
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = pack_from_f32<Tag>(v[2 * i] * rstd, v[2 * i + 1] * rstd);
        st_256(p.y + at + static_cast<int64_t>(u) * 32, o);
      } else {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = max_f32(amax, fabsf(v[i]));
        const uint32_t code = cvt_f32_to_e4m3(min_f32(__fdiv_rn(gs * (amax * rstd), 6.0f), 448.0f)) & 0xFFu;
        const float d = e4m3_to_f32(code);
        const float out_scale = d == 0.0f ? 0.0f : __fdiv_rn(gs, d) * rstd;
        float lo[8], hi[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          lo[i] = v[i] * out_scale;
          hi[i] = v[8 + i] * out_scale;
        }
        const int64_t sf_at = p.sf_pad_cols > 0 ? sf_offset_128x4(row, u, p.sf_pad_cols)
                                                : static_cast<int64_t>(row) * p.units + u;
        p.sf[sf_at] = static_cast<uint8_t>(code);
        *reinterpret_cast<uint2*>(p.y + static_cast<int64_t>(row) * (p.H >> 1) + static_cast<int64_t>(u) * 8) =
            make_uint2(cvt_e2m1x8(lo), cvt_e2m1x8(hi));
      }
    }
  }
}

template <typename Tag, int V>
int launch_gated(const GatedParams& p, bool quantize, dim3 grid, dim3 block, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (quantize) {
    B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, gated_add_rmsnorm_kernel<Tag, V, true>, p));
  } else {
    B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, gated_add_rmsnorm_kernel<Tag, V, false>, p));
  }
  return B2_OK;
}

template <typename Tag>
int dispatch_gated(const GatedParams& p, bool quantize, cudaStream_t stream) {
  // One unit per thread up to 256 units, two up to 2048 (1024 threads); a warp per row, eight rows per CTA, for short rows.
  const int per = p.units <= 256 ? 1 : 2;
  const int threads = ((p.units + per - 1) / per + 31) / 32 * 32;
  const int rows = threads == 32 ? 8 : 1;
  const dim3 grid((p.M + rows - 1) / rows), block(threads, rows);
  if (per == 1) return launch_gated<Tag, 1>(p, quantize, grid, block, stream);
  return launch_gated<Tag, 2>(p, quantize, grid, block, stream);
}

}  // namespace
}  // namespace b2

extern "C" int b2_gated_add_rmsnorm_fp4quant(const void* x, const void* residual, const void* w_post, const void* gate,
                                             const void* w_pre, void* residual_out, void* y, void* sf,
                                             const float* gs_dev, int M, int H, int rows_per_gate, float residual_scale,
                                             float eps, int in_dtype, int quantize, int swizzled, void* stream) {
  using namespace b2;
  if (in_dtype != B2_DTYPE_F16 && in_dtype != B2_DTYPE_BF16) {
    set_error("b2_gated_add_rmsnorm_fp4quant: unsupported in_dtype %d", in_dtype);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (M < 0 || H < 16 || H % 16 != 0 || H > 32768 || rows_per_gate < 1) {
    set_error("b2_gated_add_rmsnorm_fp4quant: M=%d H=%d rows_per_gate=%d: need M >= 0, H %% 16 == 0, 16 <= H <= 32768, rows_per_gate >= 1",
              M, H, rows_per_gate);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (M == 0) return B2_OK;
  if (!x || !residual || !w_pre || !residual_out || !y || (quantize && (!sf || !gs_dev))) {
    set_error("b2_gated_add_rmsnorm_fp4quant: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  const uintptr_t wide = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                         reinterpret_cast<uintptr_t>(w_post) | reinterpret_cast<uintptr_t>(gate) |
                         reinterpret_cast<uintptr_t>(w_pre) | reinterpret_cast<uintptr_t>(residual_out) |
                         (quantize ? 0 : reinterpret_cast<uintptr_t>(y));
  if ((wide & 31) || (reinterpret_cast<uintptr_t>(y) & 7) || (reinterpret_cast<uintptr_t>(gs_dev) & 3)) {
    set_error("b2_gated_add_rmsnorm_fp4quant: 16-bit tensors must be 32-byte, packed values 8-byte, the scale 4-byte aligned");
    return B2_ERR_INVALID_ARGUMENT;
  }
  GatedParams p;
  p.x = static_cast<const uint8_t*>(x);
  p.residual = static_cast<const uint8_t*>(residual);
  p.w_post = static_cast<const uint8_t*>(w_post);
  p.gate = static_cast<const uint8_t*>(gate);
  p.w_pre = static_cast<const uint8_t*>(w_pre);
  p.residual_out = static_cast<uint8_t*>(residual_out);
  p.y = static_cast<uint8_t*>(y);
  p.sf = static_cast<uint8_t*>(sf);
  p.gs = gs_dev;
  p.M = M;
  p.H = H;
  p.units = H / 16;
  p.rows_per_gate = rows_per_gate;
  p.sf_pad_cols = quantize && swizzled ? (p.units + 3) / 4 * 4 : 0;
  p.scale = residual_scale;
  p.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (in_dtype == B2_DTYPE_F16) return dispatch_gated<F16Tag>(p, quantize != 0, s);
  return dispatch_gated<BF16Tag>(p, quantize != 0, s);
}
