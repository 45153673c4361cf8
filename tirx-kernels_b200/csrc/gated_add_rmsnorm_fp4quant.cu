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
// What bounds it beside memory is instructions (32 a value at first): 16-bit factors go into mixed-precision multiply-adds
// without unpacking, pairs through f32x2, and the row's own work (two sums, two roots) is kept short.  8192 x 7168 bf16:
// 76 us, 6.2 TB/s (0.94 of the copy bandwidth); quantized 66.6 us, 5.8 TB/s (0.88); one row of 8192 3.5 us.
#include <algorithm>
#include <atomic>
#include <type_traits>

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
  float scale, eps, inv_h;
};

// Rows pass through once: kept out of L1, where the weights and the gate are to stay.
__device__ __forceinline__ void ld_256(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
__device__ __forceinline__ uint4 ld_weight_128(const void* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ void st_256(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Mixed-precision multiply-adds (sm_100): 16-bit factors, fp32 sum, no unpacking.
template <typename Tag, bool HIGH>
__device__ __forceinline__ float fma_mixed(uint32_t a, uint32_t b, float c) {
  float r;
  if constexpr (std::is_same<Tag, BF16Tag>::value) {
    if constexpr (HIGH)
      asm("{ .reg .b16 al, ah, bl, bh; mov.b32 {al, ah}, %1; mov.b32 {bl, bh}, %2; fma.rn.f32.bf16 %0, ah, bh, %3; }" : "=f"(r) : "r"(a), "r"(b), "f"(c));
    else
      asm("{ .reg .b16 al, ah, bl, bh; mov.b32 {al, ah}, %1; mov.b32 {bl, bh}, %2; fma.rn.f32.bf16 %0, al, bl, %3; }" : "=f"(r) : "r"(a), "r"(b), "f"(c));
  } else {
    if constexpr (HIGH)
      asm("{ .reg .b16 al, ah, bl, bh; mov.b32 {al, ah}, %1; mov.b32 {bl, bh}, %2; fma.rn.f32.f16 %0, ah, bh, %3; }" : "=f"(r) : "r"(a), "r"(b), "f"(c));
    else
      asm("{ .reg .b16 al, ah, bl, bh; mov.b32 {al, ah}, %1; mov.b32 {bl, bh}, %2; fma.rn.f32.f16 %0, al, bl, %3; }" : "=f"(r) : "r"(a), "r"(b), "f"(c));
  }
  return r;
}
// a^2 + sum, and the exact product (plus -0, which changes nothing, a zero's sign included).
template <typename Tag>
__device__ __forceinline__ float2 add_square(uint32_t a, float2 sum) {
  return make_float2(fma_mixed<Tag, false>(a, a, sum.x), fma_mixed<Tag, true>(a, a, sum.y));
}
template <typename Tag>
__device__ __forceinline__ float2 product(uint32_t a, uint32_t b) {
  return make_float2(fma_mixed<Tag, false>(a, b, -0.0f), fma_mixed<Tag, true>(a, b, -0.0f));
}

// Sum over the threads of a row; `red` has a slot per warp of this row.
__device__ __forceinline__ float row_sum(float v, float* red, int warps, int warp, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (warps == 1) return v;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < warps ? red[lane] : 0.0f;
  if (warps > 16) v += __shfl_xor_sync(0xffffffffu, v, 16);  // up to 8 warps: their slots are in the first eight lanes
  if (warps > 8) v += __shfl_xor_sync(0xffffffffu, v, 8);
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return __shfl_sync(0xffffffffu, v, 0);
}

// 1 / sqrt(mean + eps): the approximation and one Newton step, below one unit in the last place.  Every thread needs it
// twice a row, so correctly rounded division and root (40 instructions) would be a tenth of the kernel.
__device__ __forceinline__ float inverse_root(float sum, const GatedParams& p) {
  const float m = fmaf(sum, p.inv_h, p.eps);
  const float r = rsqrt_approx_ftz(m);
  const float better = fmaf(0.5f * r, fmaf(-m * r, r, 1.0f), r);
  return m > 0.0f && m < 1e30f ? better : r;  // zero (eps = 0), infinite and NaN rows keep 1 / sqrt's own answer
}

// One unit of y: v holds h * w_pre, exact.
template <typename Tag, bool QUANT>
__device__ __forceinline__ void store_unit(const GatedParams& p, int row, int u, const float2 (&v)[8], float rstd, float gs) {
  if constexpr (!QUANT) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = pack_pair<Tag>(mul_f32x2(v[i], make_float2(rstd, rstd)));
    st_256(p.y + (static_cast<int64_t>(row) * p.H + static_cast<int64_t>(u) * 16) * 2, o);
  } else {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_f32(amax, max_f32(fabsf(v[i].x), fabsf(v[i].y)));
    const uint32_t code = cvt_f32_to_e4m3(min_f32(gs * (amax * rstd) * (1.0f / 6.0f), 448.0f)) & 0xFFu;
    const float d = e4m3_to_f32(code);
    const float out_scale = d == 0.0f ? 0.0f : gs * rcp_approx_ftz(d) * rstd;
    const float2 o2 = make_float2(out_scale, out_scale);
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = mul_f32x2(v[i], o2), b = mul_f32x2(v[4 + i], o2);
      lo[2 * i] = a.x;
      lo[2 * i + 1] = a.y;
      hi[2 * i] = b.x;
      hi[2 * i + 1] = b.y;
    }
    const int64_t sf_at = p.sf_pad_cols > 0 ? sf_offset_128x4(row, u, p.sf_pad_cols)
                                            : static_cast<int64_t>(row) * p.units + u;
    p.sf[sf_at] = static_cast<uint8_t>(code);
    *reinterpret_cast<uint2*>(p.y + static_cast<int64_t>(row) * (p.H >> 1) + static_cast<int64_t>(u) * 8) =
        make_uint2(cvt_e2m1x8(lo), cvt_e2m1x8(hi));
  }
}

// blockDim = (threads per row, rows per CTA); more than one row per CTA only with 32 threads per row.  V units per thread.
template <typename Tag, int V, bool QUANT, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) gated_add_rmsnorm_kernel(const __grid_constant__ GatedParams p) {
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
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (t + j * static_cast<int>(blockDim.x) < p.units) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum = add_square<Tag>(x[j][i], sum);
        }
      }
    }
    rstd = inverse_root(row_sum(sum.x + sum.y, red[0], warps, warp, lane), p);
  }
  const uint8_t* gate = p.gate ? p.gate + static_cast<int64_t>(row / p.rows_per_gate) * p.H * 2 : nullptr;
  const float2 rstd2 = make_float2(rstd, rstd), scale2 = make_float2(p.scale, p.scale);
  float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int u = t + j * blockDim.x;
    if (u < p.units) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // half a unit at a time: fewer weights in registers, more rows on the SM
        uint4 w = make_uint4(0u, 0u, 0u, 0u), g = w;
        if (p.w_post) w = ld_weight_128(p.w_post + static_cast<int64_t>(u) * 32 + q * 16);
        if (gate) g = ld_weight_128(gate + static_cast<int64_t>(u) * 32 + q * 16);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w}, gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = 4 * q + k;
          float2 v = p.w_post ? mul_f32x2(product<Tag>(x[j][i], ww[k]), rstd2) : unpack2<Tag>(x[j][i]);
          if (gate) v = mul_f32x2(v, unpack2<Tag>(gw[k]));
          v = fma_f32x2(scale2, unpack2<Tag>(h[j][i]), v);
          h[j][i] = pack_pair<Tag>(v);
          sum = add_square<Tag>(h[j][i], sum);
        }
      }
      st_256(p.residual_out + at + static_cast<int64_t>(u) * 32, h[j]);
    }
  }
  rstd = inverse_root(row_sum(sum.x + sum.y, red[1], warps, warp, lane), p);
  const float gs = QUANT ? __ldg(p.gs) : 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int u = t + j * blockDim.x;
    if (u < p.units) {
      float2 v[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint4 w = ld_weight_128(p.w_pre + static_cast<int64_t>(u) * 32 + q * 16);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[4 * q + k] = product<Tag>(h[j][4 * q + k], ww[k]);
        }
      }
      store_unit<Tag, QUANT>(p, row, u, v, rstd, gs);
    }
  }
}

// Many rows.  Persistent CTAs with a ring of rows in shared memory, filled by bulk copies `stages` rows ahead: memory
// is busy while the CTA reduces and rounds, which the kernel above leaves to chance between resident rows.  A thread has
// the same columns in every row, so weights and gate stay in registers; the row's only traffic beside x, residual, h
// and y is a new gate.  x and the residual are read from the ring (x twice), h waits in registers for its norm.
constexpr int kStreamThreads = 512;
constexpr int kMaxStages = 8;
constexpr int kRingBytes = 200 * 1024;  // of an SM, shared by its CTAs

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint4 lds_128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}

static __device__ uint32_t g_gated_status;  // set when a wait for a row ran out

template <typename Tag, int V, bool QUANT>
__global__ void __launch_bounds__(kStreamThreads, V == 1 ? 2 : 1)
    gated_add_rmsnorm_stream_kernel(const __grid_constant__ GatedParams p, int stages) {
  extern __shared__ __align__(128) uint8_t ring[];  // [stages][x row, residual row]
  __shared__ __align__(8) uint64_t full[kMaxStages];
  __shared__ float red[3][32];
  __shared__ volatile int gave_up;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
  const uint32_t row_bytes = static_cast<uint32_t>(p.H) * 2;
  const uint32_t ring_at = shared_address(ring), bars = shared_address(full);
  if (t == 0) {
    for (int s = 0; s < stages; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8u * s) : "memory");
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  auto request = [&](int row, int stage) {  // thread 0
    const uint32_t bar = bars + 8u * stage, dst = ring_at + static_cast<uint32_t>(stage) * 2 * row_bytes;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * row_bytes) : "memory");
    bulk_load(dst, p.x + static_cast<int64_t>(row) * row_bytes, row_bytes, bar);
    bulk_load(dst + row_bytes, p.residual + static_cast<int64_t>(row) * row_bytes, row_bytes, bar);
  };
  if (t == 0)
    for (int s = 0; s < stages; ++s)
      if (static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(s) * gridDim.x < p.M) request(blockIdx.x + s * gridDim.x, s);

  uint4 w_post[V][2], w_pre[V][2], gate[V][2];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int u = t + j * blockDim.x;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      w_post[j][q] = w_pre[j][q] = gate[j][q] = make_uint4(0u, 0u, 0u, 0u);
      if (u < p.units) {
        if (p.w_post) w_post[j][q] = ld_weight_128(p.w_post + static_cast<int64_t>(u) * 32 + q * 16);
        w_pre[j][q] = ld_weight_128(p.w_pre + static_cast<int64_t>(u) * 32 + q * 16);
      }
    }
  }
  const float gs = QUANT ? __ldg(p.gs) : 0.0f;
  const float2 scale2 = make_float2(p.scale, p.scale);
  int64_t gate_end = 0;  // first row that needs another gate
  int stage = 0;
  uint32_t phase = 0, parity = 0;
  for (int64_t row64 = blockIdx.x; row64 < p.M; row64 += gridDim.x) {
    const int row = static_cast<int>(row64);
    const int64_t at = row64 * row_bytes;
    if (p.gate && row64 >= gate_end) {
      const int gate_row = row / p.rows_per_gate;
      gate_end = static_cast<int64_t>(gate_row + 1) * p.rows_per_gate;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int u = t + j * blockDim.x;
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (u < p.units) gate[j][q] = ld_weight_128(p.gate + static_cast<int64_t>(gate_row) * row_bytes + static_cast<int64_t>(u) * 32 + q * 16);
      }
    }
    {
      bool landed = false;
      for (uint32_t i = 0; i < (1u << 22) && !landed; ++i) landed = try_wait(bars + 8u * stage, phase);
      if (!landed) {
        gave_up = 1;
        atomicExch(&g_gated_status, 1u);
      }
    }
    const uint32_t x_at = ring_at + static_cast<uint32_t>(stage) * 2 * row_bytes;
    float rstd = 1.0f;
    if (p.w_post) {
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int u = t + j * blockDim.x;
        if (u < p.units) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint4 x = lds_128(x_at + static_cast<uint32_t>(u) * 32 + q * 16);
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              sum = add_square<Tag>(xw[k], sum);
            }
          }
        }
      }
      rstd = inverse_root(row_sum(sum.x + sum.y, red[0], warps, warp, lane), p);
    }
    const float2 rstd2 = make_float2(rstd, rstd);
    uint32_t h[V][8];
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int u = t + j * blockDim.x;
      if (u < p.units) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint4 x = lds_128(x_at + static_cast<uint32_t>(u) * 32 + q * 16);
          const uint4 r = lds_128(x_at + row_bytes + static_cast<uint32_t>(u) * 32 + q * 16);
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, rw[4] = {r.x, r.y, r.z, r.w};
          const uint32_t ww[4] = {w_post[j][q].x, w_post[j][q].y, w_post[j][q].z, w_post[j][q].w};
          const uint32_t gw[4] = {gate[j][q].x, gate[j][q].y, gate[j][q].z, gate[j][q].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float2 v = p.w_post ? mul_f32x2(product<Tag>(xw[k], ww[k]), rstd2) : unpack2<Tag>(xw[k]);
            if (p.gate) v = mul_f32x2(v, unpack2<Tag>(gw[k]));
            v = fma_f32x2(scale2, unpack2<Tag>(rw[k]), v);
            h[j][4 * q + k] = pack_pair<Tag>(v);
            sum = add_square<Tag>(h[j][4 * q + k], sum);
          }
        }
        st_256(p.residual_out + at + static_cast<int64_t>(u) * 32, h[j]);
      }
    }
    // The second sum's barrier also says that every thread is done with this stage (its buffer alternates: without a
    // first sum nothing else stands between two rows).
    rstd = inverse_root(row_sum(sum.x + sum.y, red[1 + parity], warps, warp, lane), p);
    parity ^= 1u;
    if (gave_up) break;
    if (t == 0 && row64 + static_cast<int64_t>(stages) * gridDim.x < p.M) request(row + stages * static_cast<int>(gridDim.x), stage);
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int u = t + j * blockDim.x;
      if (u < p.units) {
        float2 v[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t ww[4] = {w_pre[j][q].x, w_pre[j][q].y, w_pre[j][q].z, w_pre[j][q].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) v[4 * q + k] = product<Tag>(h[j][4 * q + k], ww[k]);
        }
        store_unit<Tag, QUANT>(p, row, u, v, rstd, gs);
      }
    }
  }
  if (gave_up)
    for (int i = 0; i < 64; ++i) __nanosleep(2000);  // copies that are still on their way land before the memory goes
}

template <typename Tag, int V, int THREADS, int BLOCKS>
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
    B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, gated_add_rmsnorm_kernel<Tag, V, true, THREADS, BLOCKS>, p));
  } else {
    B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, gated_add_rmsnorm_kernel<Tag, V, false, THREADS, BLOCKS>, p));
  }
  return B2_OK;
}

template <typename Tag, int V, bool QUANT>
int launch_stream(const GatedParams& p, int threads, int per_sm, int stages, int sms, cudaStream_t stream) {
  auto kernel = gated_add_rmsnorm_stream_kernel<Tag, V, QUANT>;
  {
    static std::atomic<bool> configured[64] = {};  // setting it twice does no harm
    int dev = 0;
    B2_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      B2_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(per_sm * sms);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(stages) * 4 * p.H;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p, stages));
  return B2_OK;
}

template <typename Tag>
int dispatch_gated(const GatedParams& p, bool quantize, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (sms <= 0) return B2_ERR_CUDA;
  // The ring, for many rows, where it wins: quantized (8192 x 7168: 66.6 us for 72.1 by the kernel without it) and rows of
  // more than 8192 (4096 x 16384: 102 for 107, quantized 91 for 101), not 16-bit rows below that (8192 x 7168: 77 to 85 for 76;
  // 8192 x 4096: 55 for 52).  Rows of 33 to 1024 units, one per thread (two above 512), as many CTAs as 1024 threads make (one, of
  // 512, where a thread has two units), and at least two rows ahead and four rows for every CTA.
  if (p.units > 32 && p.units <= 1024 && (quantize || p.units > kStreamThreads)) {
    const int per = p.units <= kStreamThreads ? 1 : 2;
    const int threads = ((p.units + per - 1) / per + 31) / 32 * 32;
    int per_sm = per == 1 ? 1024 / threads : 1;
    const int row = 4 * p.H;
    while (per_sm > 1 && kRingBytes / per_sm / row < 2) --per_sm;
    const int stages = std::min(kMaxStages, kRingBytes / per_sm / row);
    if (stages >= 2 && p.M >= 4 * per_sm * sms) {
      if (per == 1)
        return quantize ? launch_stream<Tag, 1, true>(p, threads, per_sm, stages, sms, stream)
                        : launch_stream<Tag, 1, false>(p, threads, per_sm, stages, sms, stream);
      return quantize ? launch_stream<Tag, 2, true>(p, threads, per_sm, stages, sms, stream)
                      : launch_stream<Tag, 2, false>(p, threads, per_sm, stages, sms, stream);
    }
  }
  // One unit per thread up to 256 units, two up to 2048 (1024 threads); a warp per row, eight rows per CTA, for short rows.
  const int per = p.units <= 256 ? 1 : 2;
  const int threads = ((p.units + per - 1) / per + 31) / 32 * 32;
  const int rows = threads == 32 ? 8 : 1;
  const dim3 grid((p.M + rows - 1) / rows), block(threads, rows);
  if (per == 1) return launch_gated<Tag, 1, 256, 6>(p, quantize, grid, block, stream);
  if (threads <= 256) return launch_gated<Tag, 2, 256, 4>(p, quantize, grid, block, stream);
  return launch_gated<Tag, 2, 1024, 1>(p, quantize, grid, block, stream);
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
  p.inv_h = 1.0f / static_cast<float>(H);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (in_dtype == B2_DTYPE_F16) return dispatch_gated<F16Tag>(p, quantize != 0, s);
  return dispatch_gated<BF16Tag>(p, quantize != 0, s);
}

extern "C" int b2_gated_add_rmsnorm_fp4quant_status(void* stream) {
  using namespace b2;
  void* word = nullptr;
  B2_CUDA_TRY(cudaGetSymbolAddress(&word, g_gated_status));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t host = 0;
  B2_CUDA_TRY(cudaMemcpyAsync(&host, word, sizeof(host), cudaMemcpyDeviceToHost, s));
  B2_CUDA_TRY(cudaStreamSynchronize(s));
  if (host == 0) return B2_OK;
  B2_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(host), s));
  set_error("b2_gated_add_rmsnorm_fp4quant: the wait for a row ran out");
  return B2_ERR_DEVICE_TIMEOUT;
}
