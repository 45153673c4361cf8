// The routed feed-forward around the grouped product (nvfp4_grouped_gemm.cu): routing plan, quantizer with the
// grouped scale layout, weighted sum per token, and the whole of it as one call, for sm_100a.
//
//   plan      assignment i = (token i / topk, expert ids[i]) gets row position[i]; rows are sorted by expert, within an
//             expert by assignment (a stable counting sort: no atomics, the same rows on every run)
//   quantize  row r of the output is row index[r] of the input, in NVFP4 with the encode scale of r's group, its scale
//             factors in the 128 x 4 tiles of that group (first tile offsets[g] / 128 + g)
//   combine   out[t] = residual[t] + sum over k of weight[t, k] * y[position[t, k]], in order of k, fp32, one rounding
#include <algorithm>
#include <atomic>

#include "quant_block.cuh"

namespace b2 {
namespace {

constexpr int kMaxGroups = 384;  // as in nvfp4_grouped_gemm.cu

template <typename... Params>
int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                     Params... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return B2_OK;
}

// ---- plan ----------------------------------------------------------------------------------------
constexpr int kPlanWarps = 32;

// One CTA.  Every warp has a run of consecutive assignments and a histogram of its own; a scan over warps and experts
// turns the histograms into first rows, and a second walk over the same run hands the rows out in order.
__global__ void __launch_bounds__(kPlanWarps * 32)
    moe_plan_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ offsets, int32_t* __restrict__ row_token,
                    int32_t* __restrict__ position, int n, int topk, int experts) {
  extern __shared__ int hist[];  // [kPlanWarps][experts]
  __shared__ int start[kMaxGroups + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  int* mine = hist + warp * experts;
  for (int e = lane; e < experts; e += 32) mine[e] = 0;
  __syncwarp();
  const int run = ((n + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int64_t first64 = static_cast<int64_t>(warp) * run;
  const int first = static_cast<int>(first64 < n ? first64 : n), last = static_cast<int>(first64 + run < n ? first64 + run : n);
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    int id = i < last ? ids[i] : -1;
    if (id < 0 || id >= experts) id = -1;  // dropped
    const unsigned peers = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && lane == __ffs(peers) - 1) mine[id] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int sum = 0;
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = hist[w * experts + e];
      hist[w * experts + e] = sum;
      sum += c;
    }
    start[e] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int before = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + lane;
      const int count = e < experts ? start[e] : 0;
      int sum = count;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (e < experts) {
        start[e] = before + sum - count;
        offsets[e] = before + sum - count;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
      start[experts] = before;
      offsets[experts] = before;
    }
  }
  __syncthreads();
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    int id = i < last ? ids[i] : -1;
    if (id < 0 || id >= experts) id = -1;
    const unsigned peers = __match_any_sync(0xffffffffu, id);
    int row = -1;
    if (id >= 0) row = start[id] + mine[id] + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (id >= 0 && lane == __ffs(peers) - 1) mine[id] += __popc(peers);
    __syncwarp();
    if (i < last) position[i] = row;
    if (row >= 0) row_token[row] = i / topk;
  }
  for (int r = start[experts] + threadIdx.x; r < n; r += blockDim.x) row_token[r] = -1;
}

// ---- quantizer with the grouped scale layout -------------------------------------------------------
struct GroupedQuantParams {
  const uint8_t* in;       // [in_rows, k] ([in_rows, 2k] with SILU)
  const int32_t* index;    // [rows] or null: row r of the input
  const int32_t* offsets;  // [groups + 1]
  uint8_t* out;            // [rows, k / 2]
  uint8_t* sf;
  const float* gs;         // [groups]
  int in_rows, rows, groups, k;
};

constexpr int kQuantThreads = 128;

// One CTA per row.  Thread t has blocks t, t + 128, ...; up to UNROLL of them are loaded before the first is used, and
// the row's group is looked up while they are on their way.
template <typename Tag, bool SILU, bool V8, int UNROLL>
__global__ void __launch_bounds__(kQuantThreads) nvfp4_quantize_grouped_kernel(const __grid_constant__ GroupedQuantParams p) {
  const int row = blockIdx.x;
  const int t = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  if (row >= __ldg(p.offsets + p.groups)) return;  // behind the last group: left as it was
  const int source = p.index ? __ldg(p.index + row) : row;
  const bool there = source >= 0 && source < p.in_rows;  // a row that does not exist is quantized as zeros
  const int nsb = p.k / 16;
  const uint8_t* in_row = p.in + static_cast<int64_t>(there ? source : 0) * p.k * (SILU ? 4 : 2);
  uint8_t* out_row = p.out + static_cast<int64_t>(row) * (p.k >> 1);
  float gs = 0.0f, rcp_gs = 0.0f;
  int sf_row = -1;
  const float rcp6 = rcp_approx_ftz(6.0f);
  for (int c0 = t; c0 < nsb; c0 += kQuantThreads * UNROLL) {
    uint32_t w[UNROLL][8];
    uint32_t u[SILU ? UNROLL : 1][8];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int col = c0 + j * kQuantThreads;
      if (there && col < nsb) {
        load_block<V8>(in_row + col * 32, w[j]);
        if constexpr (SILU) load_block<V8>(in_row + 2 * static_cast<int64_t>(p.k) + col * 32, u[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[j][i] = 0u;
        if constexpr (SILU) {
#pragma unroll
          for (int i = 0; i < 8; ++i) u[j][i] = 0u;
        }
      }
    }
    if (sf_row < 0) {
      int lo = 0, hi = p.groups;  // the last group that begins at or in front of the row
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.offsets + mid) <= row) lo = mid;
        else hi = mid;
      }
      const int first = min(max(__ldg(p.offsets + lo), 0), row);  // bad offsets stay inside the buffer
      sf_row = ((first >> 7) + lo) * 128 + row - first;
      gs = __ldg(p.gs + lo);
      rcp_gs = rcp_approx_ftz(gs);
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int col = c0 + j * kQuantThreads;
      if (col >= nsb) break;
      if constexpr (SILU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[j][i] = silu_and_mul_pair<Tag>(w[j][i], u[j][i]);
      }
      uint32_t sf_byte;
      uint2 packed;
      quantize_block<Tag>(w[j], gs, rcp_gs, rcp6, sf_byte, packed);
      p.sf[sf_offset_128x4(sf_row, col, nsb)] = static_cast<uint8_t>(sf_byte);
      *reinterpret_cast<uint2*>(out_row + col * 8) = packed;
    }
  }
}

template <typename Tag, bool SILU>
int launch_quantize(const GroupedQuantParams& p, bool v8, cudaStream_t s) {
  constexpr int kUnroll = SILU ? 1 : 2;
  const dim3 grid(p.rows);
  if (v8) return launch_dependent(nvfp4_quantize_grouped_kernel<Tag, SILU, true, kUnroll>, grid, kQuantThreads, 0, s, p);
  return launch_dependent(nvfp4_quantize_grouped_kernel<Tag, SILU, false, kUnroll>, grid, kQuantThreads, 0, s, p);
}

// ---- weighted sum per token --------------------------------------------------------------------------
struct CombineParams {
  const uint16_t* y;        // [rows, n]
  const int32_t* position;  // [tokens, topk]
  const float* weight;      // [tokens, topk]
  const uint16_t* residual; // [tokens, n] or null
  uint16_t* out;            // [tokens, n]
  int rows, tokens, topk, n;
  int parts;                // CTAs per token
};

constexpr int kCombineThreads = 128;

// One CTA per token and 1024 columns, 8 columns per thread.  Positions outside [0, rows) (dropped assignments) add nothing.
template <typename Tag>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(const __grid_constant__ CombineParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int token = blockIdx.x / p.parts;
  const int col = ((blockIdx.x % p.parts) * kCombineThreads + static_cast<int>(threadIdx.x)) * 8;
  if (col >= p.n) return;
  const int64_t at = static_cast<int64_t>(token) * p.n + col;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  if (p.residual) {
    uint32_t r[4];
    ld_stream_128(p.residual + at, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<Tag>(r[i]);
      acc[2 * i] = f.x;
      acc[2 * i + 1] = f.y;
    }
  }
  const int32_t* position = p.position + static_cast<int64_t>(token) * p.topk;
  const float* weight = p.weight + static_cast<int64_t>(token) * p.topk;
  for (int k0 = 0; k0 < p.topk; k0 += 4) {
    uint32_t r[4][4];
    float w[4];
    bool live[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pos = k0 + j < p.topk ? __ldg(position + k0 + j) : -1;
      live[j] = pos >= 0 && pos < p.rows;
      if (live[j]) {
        w[j] = __ldg(weight + k0 + j);
        ld_stream_128(p.y + static_cast<int64_t>(pos) * p.n + col, r[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!live[j]) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<Tag>(r[j][i]);
        acc[2 * i] = fmaf(w[j], f.x, acc[2 * i]);
        acc[2 * i + 1] = fmaf(w[j], f.y, acc[2 * i + 1]);
      }
    }
  }
  *reinterpret_cast<uint4*>(p.out + at) =
      make_uint4(pack_from_f32<Tag>(acc[0], acc[1]), pack_from_f32<Tag>(acc[2], acc[3]),
                 pack_from_f32<Tag>(acc[4], acc[5]), pack_from_f32<Tag>(acc[6], acc[7]));
}

bool misaligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace
}  // namespace b2

extern "C" int b2_moe_plan(const int32_t* ids_dev, int32_t* offsets_dev, int32_t* row_token_dev, int32_t* position_dev,
                           int tokens, int topk, int experts, void* stream) {
  using namespace b2;
  if (tokens < 0 || topk < 1 || experts < 1 || experts > kMaxGroups || static_cast<int64_t>(tokens) * topk > 0x7fffffff - 1024) {
    set_error("b2_moe_plan: tokens=%d topk=%d experts=%d: need tokens >= 0, topk >= 1, 1 to %d experts, below 2^31 assignments",
              tokens, topk, experts, kMaxGroups);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (!offsets_dev || (tokens > 0 && (!ids_dev || !row_token_dev || !position_dev))) {
    set_error("b2_moe_plan: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (misaligned(ids_dev, 4) || misaligned(offsets_dev, 4) || misaligned(row_token_dev, 4) || misaligned(position_dev, 4)) {
    set_error("b2_moe_plan: all tensors must be 4-byte aligned");
    return B2_ERR_INVALID_ARGUMENT;
  }
  const size_t smem = static_cast<size_t>(kPlanWarps) * experts * 4;
  {
    static std::atomic<bool> configured[64] = {};
    int dev = 0;
    B2_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      B2_CUDA_TRY(cudaFuncSetAttribute(moe_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanWarps * kMaxGroups * 4));
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
  }
  return launch_dependent(moe_plan_kernel, dim3(1), kPlanWarps * 32, smem, static_cast<cudaStream_t>(stream), ids_dev,
                          offsets_dev, row_token_dev, position_dev, tokens * topk, topk, experts);
}

extern "C" int64_t b2_nvfp4_grouped_sf_bytes(int rows, int groups, int k) {
  if (rows < 0 || groups < 1 || groups > b2::kMaxGroups || k <= 0 || k % 64 != 0) return -1;
  return (static_cast<int64_t>(rows / 128) + groups) * 128 * (k / 16);
}

extern "C" int b2_nvfp4_quantize_grouped(const void* in, const int32_t* index_dev, const int32_t* offsets_dev, void* out,
                                         void* sf, const float* gs_dev, int in_rows, int rows, int groups, int k,
                                         int in_dtype, int fuse_silu, void* stream) {
  using namespace b2;
  if (in_dtype != B2_DTYPE_F16 && in_dtype != B2_DTYPE_BF16) {
    set_error("b2_nvfp4_quantize_grouped: unsupported in_dtype %d", in_dtype);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (rows < 0 || rows > 0x7fffffff - 512 || in_rows < 0 || groups < 1 || groups > kMaxGroups || k < 64 || k % 64 != 0 ||
      k > (1 << 28) || static_cast<int64_t>(rows) + 128 * (groups + 1) > 0x7fffffffll) {
    set_error("b2_nvfp4_quantize_grouped: in_rows=%d rows=%d groups=%d k=%d: need rows >= 0, 1 to %d groups, k %% 64 == 0",
              in_rows, rows, groups, k, kMaxGroups);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (!index_dev && in_rows < rows) {
    set_error("b2_nvfp4_quantize_grouped: %d input rows for %d rows without an index", in_rows, rows);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (rows == 0) return B2_OK;
  if (!in || !offsets_dev || !out || !sf || !gs_dev) {
    set_error("b2_nvfp4_quantize_grouped: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (misaligned(in, 16) || misaligned(out, 8) || misaligned(index_dev, 4) || misaligned(offsets_dev, 4) || misaligned(gs_dev, 4)) {
    set_error("b2_nvfp4_quantize_grouped: `in` must be 16-byte, `out` 8-byte, index, offsets and scales 4-byte aligned");
    return B2_ERR_INVALID_ARGUMENT;
  }
  GroupedQuantParams p;
  p.in = static_cast<const uint8_t*>(in);
  p.index = index_dev;
  p.offsets = offsets_dev;
  p.out = static_cast<uint8_t*>(out);
  p.sf = static_cast<uint8_t*>(sf);
  p.gs = gs_dev;
  p.in_rows = in_rows;
  p.rows = rows;
  p.groups = groups;
  p.k = k;
  const bool v8 = !misaligned(in, 32);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (in_dtype == B2_DTYPE_F16)
    return fuse_silu ? launch_quantize<F16Tag, true>(p, v8, s) : launch_quantize<F16Tag, false>(p, v8, s);
  return fuse_silu ? launch_quantize<BF16Tag, true>(p, v8, s) : launch_quantize<BF16Tag, false>(p, v8, s);
}

extern "C" int b2_moe_combine(const void* y, const int32_t* position_dev, const float* weight_dev, const void* residual,
                              void* out, int rows, int tokens, int topk, int n, int dtype, void* stream) {
  using namespace b2;
  if (dtype != B2_DTYPE_F16 && dtype != B2_DTYPE_BF16) {
    set_error("b2_moe_combine: unsupported dtype %d", dtype);
    return B2_ERR_INVALID_ARGUMENT;
  }
  const int64_t parts = (static_cast<int64_t>(n) + kCombineThreads * 8 - 1) / (kCombineThreads * 8);
  if (rows < 0 || tokens < 0 || topk < 1 || n < 1 || n % 8 != 0 || parts * tokens > 0x7fffffffll) {
    set_error("b2_moe_combine: rows=%d tokens=%d topk=%d n=%d: need rows, tokens >= 0, topk >= 1, n %% 8 == 0", rows, tokens, topk, n);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (tokens == 0) return B2_OK;
  if ((rows > 0 && !y) || !position_dev || !weight_dev || !out) {
    set_error("b2_moe_combine: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (misaligned(y, 16) || misaligned(out, 16) || misaligned(residual, 16) || misaligned(position_dev, 4) || misaligned(weight_dev, 4)) {
    set_error("b2_moe_combine: y, residual and out must be 16-byte, position and weight 4-byte aligned");
    return B2_ERR_INVALID_ARGUMENT;
  }
  CombineParams p;
  p.y = static_cast<const uint16_t*>(y);
  p.position = position_dev;
  p.weight = weight_dev;
  p.residual = static_cast<const uint16_t*>(residual);
  p.out = static_cast<uint16_t*>(out);
  p.rows = rows;
  p.tokens = tokens;
  p.topk = topk;
  p.n = n;
  p.parts = static_cast<int>(parts);
  const dim3 grid(static_cast<unsigned>(parts * tokens));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == B2_DTYPE_F16) return launch_dependent(moe_combine_kernel<F16Tag>, grid, kCombineThreads, 0, s, p);
  return launch_dependent(moe_combine_kernel<BF16Tag>, grid, kCombineThreads, 0, s, p);
}

// ---- the routed feed-forward as one call ---------------------------------------------------------------
namespace b2 {
namespace {

// Workspace of b2_moe_expert_ffn: every part begins on a 256-byte boundary.
struct FfnWorkspace {
  int64_t offsets, row_token, position, a1, sf1, y1, a2, sf2, z, total;
};
FfnWorkspace ffn_workspace(int64_t tokens, int64_t topk, int64_t experts, int64_t hidden, int64_t inner) {
  FfnWorkspace w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const int64_t rows = tokens * topk, tiles = rows / 128 + experts;
  w.offsets = take((experts + 1) * 4);
  w.row_token = take(rows * 4);
  w.position = take(rows * 4);
  w.a1 = take(rows * (hidden / 2));
  w.sf1 = take(tiles * 128 * (hidden / 16));
  w.y1 = take(rows * inner * 4);
  w.a2 = take(rows * (inner / 2));
  w.sf2 = take(tiles * 128 * (inner / 16));
  w.z = take(rows * hidden * 2);
  w.total = at;
  return w;
}
bool ffn_sizes_ok(int tokens, int topk, int experts, int hidden, int inner) {
  return tokens >= 0 && topk >= 1 && experts >= 1 && experts <= kMaxGroups && hidden >= 64 && hidden % 64 == 0 &&
         hidden <= (1 << 24) && inner >= 64 && inner % 64 == 0 && inner <= (1 << 24) &&
         static_cast<int64_t>(tokens) * topk <= 0x7fffffff - 65536;
}

}  // namespace
}  // namespace b2

extern "C" int64_t b2_moe_expert_ffn_workspace_bytes(int tokens, int topk, int experts, int hidden, int inner) {
  if (!b2::ffn_sizes_ok(tokens, topk, experts, hidden, inner)) return -1;
  return b2::ffn_workspace(tokens, topk, experts, hidden, inner).total;
}

extern "C" int b2_moe_expert_ffn(const void* x, const int32_t* ids_dev, const float* weight_dev, const void* W1,
                                 const void* SF1, const float* alpha1_dev, const float* gs1_dev, const void* W2,
                                 const void* SF2, const float* alpha2_dev, const float* gs2_dev, const void* residual,
                                 void* out, void* workspace, int64_t workspace_bytes, int tokens, int topk, int experts,
                                 int hidden, int inner, int dtype, void* stream) {
  using namespace b2;
  if (!ffn_sizes_ok(tokens, topk, experts, hidden, inner)) {
    set_error("b2_moe_expert_ffn: tokens=%d topk=%d experts=%d hidden=%d inner=%d: need tokens >= 0, topk >= 1, 1 to %d experts, "
              "hidden %% 64 == 0, inner %% 64 == 0", tokens, topk, experts, hidden, inner, kMaxGroups);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (dtype != B2_DTYPE_F16 && dtype != B2_DTYPE_BF16) {
    set_error("b2_moe_expert_ffn: unsupported dtype %d", dtype);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (tokens == 0) return B2_OK;
  const FfnWorkspace w = ffn_workspace(tokens, topk, experts, hidden, inner);
  if (!workspace || workspace_bytes < w.total || misaligned(workspace, 256)) {
    set_error("b2_moe_expert_ffn: workspace of %lld bytes, aligned to 256, needed, %lld given", static_cast<long long>(w.total),
              static_cast<long long>(workspace ? workspace_bytes : 0));
    return B2_ERR_INVALID_ARGUMENT;
  }
  uint8_t* base = static_cast<uint8_t*>(workspace);
  int32_t* offsets = reinterpret_cast<int32_t*>(base + w.offsets);
  int32_t* row_token = reinterpret_cast<int32_t*>(base + w.row_token);
  int32_t* position = reinterpret_cast<int32_t*>(base + w.position);
  const int rows = tokens * topk;
  // Every argument is checked before the first launch: a refused call leaves nothing half done.
  if (!x || !ids_dev || !weight_dev || !W1 || !SF1 || !alpha1_dev || !gs1_dev || !W2 || !SF2 || !alpha2_dev || !gs2_dev || !out) {
    set_error("b2_moe_expert_ffn: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (misaligned(x, 16) || misaligned(W1, 16) || misaligned(SF1, 16) || misaligned(W2, 16) || misaligned(SF2, 16) ||
      misaligned(residual, 16) || misaligned(out, 16) || misaligned(ids_dev, 4) || misaligned(weight_dev, 4) ||
      misaligned(alpha1_dev, 4) || misaligned(gs1_dev, 4) || misaligned(alpha2_dev, 4) || misaligned(gs2_dev, 4)) {
    set_error("b2_moe_expert_ffn: activations, weights and their scales must be 16-byte aligned, all else 4-byte");
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (static_cast<int64_t>(experts) * ((2 * inner + 127) / 128 * 128) > 0x7fffffffll ||
      static_cast<int64_t>(experts) * ((hidden + 127) / 128 * 128) > 0x7fffffffll) {
    set_error("b2_moe_expert_ffn: experts=%d of hidden=%d, inner=%d: the weights' rows exceed 2^31", experts, hidden, inner);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (int rc = b2_moe_plan(ids_dev, offsets, row_token, position, tokens, topk, experts, stream)) return rc;
  if (int rc = b2_nvfp4_quantize_grouped(x, row_token, offsets, base + w.a1, base + w.sf1, gs1_dev, tokens, rows, experts,
                                         hidden, dtype, 0, stream))
    return rc;
  if (int rc = b2_nvfp4_grouped_gemm(base + w.a1, W1, base + w.sf1, SF1, alpha1_dev, offsets, nullptr, base + w.y1, rows,
                                     experts, 2 * inner, hidden, dtype, B2_ACT_NONE, stream))
    return rc;
  if (int rc = b2_nvfp4_quantize_grouped(base + w.y1, nullptr, offsets, base + w.a2, base + w.sf2, gs2_dev, rows, rows,
                                         experts, inner, dtype, 1, stream))
    return rc;
  if (int rc = b2_nvfp4_grouped_gemm(base + w.a2, W2, base + w.sf2, SF2, alpha2_dev, offsets, nullptr, base + w.z, rows,
                                     experts, hidden, inner, dtype, B2_ACT_NONE, stream))
    return rc;
  return b2_moe_combine(base + w.z, position, weight_dev, residual, out, rows, tokens, topk, hidden, dtype, stream);
}
