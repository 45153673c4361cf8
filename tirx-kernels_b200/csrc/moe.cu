// The routed feed-forward around the grouped product (nvfp4_grouped_gemm.cu): routing plan, quantizer with the
// grouped scale layout, weighted sum per token, and the whole of it as one call, for sm_100a.
//
//   plan      assignment i = (token i / topk, expert ids[i]) gets row position[i]; rows are sorted by expert, within an
//             expert by assignment (a stable counting sort: no atomics, the same rows on every run)
//   dispatch  every token's row, read once, is quantized for each of its experts into the row that the plan gave it (the
//             same blocks where the encode scales are the same); a few assignments are planned in the same launch
//   quantize  row r of the output is row index[r] of the input, in NVFP4 with the encode scale of r's group, its scale
//             factors in the 128 x 4 tiles of that group (first tile offsets[g] / 128 + g)
//   combine   out[t] = residual[t] + sum over k of weight[t, k] * y[position[t, k]], in order of k, fp32, one rounding
#include <algorithm>
#include <atomic>

#include "quant_block.cuh"

namespace b2 {

// nvfp4_grouped_gemm.cu
int grouped_product(const void* A, const void* B, const void* SFA, const void* SFB, const float* alpha_dev,
                    const int32_t* offsets_dev, const void* bias, void* D, int rows, int groups, int N, int K,
                    int out_dtype, int activation, bool early, const int32_t* ids_dev, void* stream);
int grouped_product_gated(const void* A, const void* B, const void* SFA, const void* SFB, const float* alpha_dev,
                          const int32_t* offsets_dev, const float* gs_dev, void* out, void* sf, int rows, int groups,
                          int inner, int K, int dtype, bool early, const int32_t* ids_dev, void* stream);

namespace {

constexpr int kMaxGroups = 384;  // as in nvfp4_grouped_gemm.cu

template <typename... Params>
int launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 threads, size_t smem, cudaStream_t stream,
                     Params... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
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

constexpr int kPlanAhead = 16;

// Assignments at, at + 32, ...; what is behind the run or names no expert is -1.
__device__ __forceinline__ void load_ids(const int32_t* __restrict__ ids, int at, int last, int experts, int (&id)[kPlanAhead]) {
#pragma unroll
  for (int j = 0; j < kPlanAhead; ++j) id[j] = at + 32 * j < last ? __ldg(ids + at + 32 * j) : -1;
#pragma unroll
  for (int j = 0; j < kPlanAhead; ++j)
    if (id[j] < 0 || id[j] >= experts) id[j] = -1;
}

// Lanes with the same id (-1 among them), by a ballot per bit: __match_any_sync goes through the distinct ids one by one
// and took 24 us for 16384 assignments.
__device__ __forceinline__ unsigned same_id(int id, int bits) {
  unsigned peers = __ballot_sync(0xffffffffu, id < 0);
  if (id >= 0) peers = ~peers;
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, id >> b & 1);
    peers &= id >> b & 1 ? set : ~set;
  }
  return peers;
}

// Exclusive sums of count[0 .. experts) by one warp: start[e], and the total behind the last.
__device__ __forceinline__ void scan_experts(int* start, int experts, int lane) {
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
    if (e < experts) start[e] = before + sum - count;
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) start[experts] = before;
}

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
  const int bits = 32 - __clz(experts);
  int id[kPlanAhead];  // loads ahead of their use
  for (int i0 = first; i0 < last; i0 += 32 * kPlanAhead) {
    load_ids(ids, i0 + lane, last, experts, id);
#pragma unroll
    for (int j = 0; j < kPlanAhead; ++j) {
      if (i0 + 32 * j >= last) break;
      const unsigned peers = same_id(id[j], bits);
      if (id[j] >= 0 && lane == __ffs(peers) - 1) mine[id[j]] += __popc(peers);
      __syncwarp();
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int c[kPlanWarps], sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) c[w] = hist[w * experts + e];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      hist[w * experts + e] = sum;
      sum += c[w];
    }
    start[e] = sum;
  }
  __syncthreads();
  if (warp == 0) scan_experts(start, experts, lane);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = start[e];
  const bool again = last - first > 32 * kPlanAhead;  // else the ids are still in registers
  for (int i0 = first; i0 < last; i0 += 32 * kPlanAhead) {
    if (again) load_ids(ids, i0 + lane, last, experts, id);
#pragma unroll
    for (int j = 0; j < kPlanAhead; ++j) {
      const int i = i0 + 32 * j + lane;
      if (i0 + 32 * j >= last) break;
      const unsigned peers = same_id(id[j], bits);
      int row = -1;
      if (id[j] >= 0) row = start[id[j]] + mine[id[j]] + __popc(peers & ((1u << lane) - 1u));
      __syncwarp();
      if (id[j] >= 0 && lane == __ffs(peers) - 1) mine[id[j]] += __popc(peers);
      __syncwarp();
      if (i < last) position[i] = row;
      if (row >= 0) row_token[row] = i / topk;
    }
  }
  for (int r = start[experts] + threadIdx.x; r < n; r += blockDim.x) row_token[r] = -1;
}

// The same plan by many CTAs of 1024 assignments each, without row_token: counts per CTA, then every CTA adds up what
// the others have in front of it.  16384 assignments: 21 us by one CTA (half of it the scattered row_token), 5 by these.
constexpr int kPlanBlock = kPlanWarps * 32;
__global__ void __launch_bounds__(kPlanBlock) moe_count_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ counts,
                                                               int n, int experts) {
  __shared__ int hist[kMaxGroups];
  pdl_wait();
  pdl_launch_dependents();
  for (int e = threadIdx.x; e < experts; e += kPlanBlock) hist[e] = 0;
  __syncthreads();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kPlanBlock + threadIdx.x;
  const int id = i < n ? __ldg(ids + i) : -1;
  if (id >= 0 && id < experts) atomicAdd(hist + id, 1);  // integers: no order to matter
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kPlanBlock) counts[static_cast<int64_t>(blockIdx.x) * experts + e] = hist[e];
}
__global__ void __launch_bounds__(kPlanBlock)
    moe_rank_kernel(const int32_t* __restrict__ ids, const int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                    int32_t* __restrict__ position, int n, int experts) {
  extern __shared__ int hist[];  // [kPlanWarps][experts]: this CTA's assignments of an expert in front of a warp
  __shared__ int start[kMaxGroups + 1], ahead[kMaxGroups];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  for (int j = threadIdx.x; j < kPlanWarps * experts; j += kPlanBlock) hist[j] = 0;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kPlanBlock + threadIdx.x;
  int id = i < n ? __ldg(ids + i) : -1;
  if (id < 0 || id >= experts) id = -1;
  __syncthreads();
  const unsigned peers = same_id(id, 32 - __clz(experts));
  if (id >= 0 && lane == __ffs(peers) - 1) hist[warp * experts + id] = __popc(peers);
  for (int e = threadIdx.x; e < experts; e += kPlanBlock) {
    int total = 0, before = 0;
#pragma unroll 8
    for (int b = 0; b < static_cast<int>(gridDim.x); ++b) {
      const int c = __ldg(counts + static_cast<int64_t>(b) * experts + e);
      total += c;
      if (b < static_cast<int>(blockIdx.x)) before += c;
    }
    start[e] = total;
    ahead[e] = before;
  }
  __syncthreads();
  if (warp == 0) scan_experts(start, experts, lane);
  for (int e = threadIdx.x; e < experts; e += kPlanBlock) {
    int c[kPlanWarps], sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) c[w] = hist[w * experts + e];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      hist[w * experts + e] = sum;
      sum += c[w];
    }
  }
  __syncthreads();
  if (i < n)
    position[i] = id < 0 ? -1 : start[id] + ahead[id] + hist[warp * experts + id] + __popc(peers & ((1u << lane) - 1u));
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= experts; e += kPlanBlock) offsets[e] = start[e];
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

constexpr int kQuantThreads = 256;  // most threads of a CTA

// blockDim = (threads of a row, rows).  Thread t of a row has blocks t, t + threads, ...; up to UNROLL of them are loaded
// before the first is used, and the row's group is looked up while they are on their way.
template <typename Tag, bool SILU, bool V8, int UNROLL>
__global__ void __launch_bounds__(kQuantThreads) nvfp4_quantize_grouped_kernel(const __grid_constant__ GroupedQuantParams p) {
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int t = threadIdx.x;
  const int threads = blockDim.x;
  pdl_wait();
  pdl_launch_dependents();
  if (row >= p.rows || row >= __ldg(p.offsets + p.groups)) return;  // behind the last group: left as it was
  const int source = p.index ? __ldg(p.index + row) : row;
  const bool there = source >= 0 && source < p.in_rows;  // a row that does not exist is quantized as zeros
  const int nsb = p.k / 16;
  const uint8_t* in_row = p.in + static_cast<int64_t>(there ? source : 0) * p.k * (SILU ? 4 : 2);
  uint8_t* out_row = p.out + static_cast<int64_t>(row) * (p.k >> 1);
  float gs = 0.0f, rcp_gs = 0.0f;
  int sf_row = -1;
  const float rcp6 = rcp_approx_ftz(6.0f);
  for (int c0 = t; c0 < nsb; c0 += threads * UNROLL) {
    uint32_t w[UNROLL][8];
    uint32_t u[SILU ? UNROLL : 1][8];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int col = c0 + j * threads;
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
      const int col = c0 + j * threads;
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

// Threads of a row: as few passes over its blocks as 128 threads allow, in whole warps; rows to fill a CTA of 256.
void row_geometry(int nsb, int rows, dim3& block, dim3& grid) {
  const int passes = (nsb + 127) / 128;
  const int threads = ((nsb + passes - 1) / passes + 31) / 32 * 32;
  const int per = std::max(1, std::min(kQuantThreads / threads, rows));
  block = dim3(threads, per);
  grid = dim3((rows + per - 1) / per);
}

template <typename Tag, bool SILU>
int launch_quantize(const GroupedQuantParams& p, bool v8, cudaStream_t s) {
  constexpr int kUnroll = SILU ? 1 : 2;
  dim3 block, grid;
  row_geometry(p.k / 16, p.rows, block, grid);
  if (v8) return launch_dependent(nvfp4_quantize_grouped_kernel<Tag, SILU, true, kUnroll>, grid, block, 0, s, p);
  return launch_dependent(nvfp4_quantize_grouped_kernel<Tag, SILU, false, kUnroll>, grid, block, 0, s, p);
}

// ---- quantizer from a token to all of its experts ----------------------------------------------------------
struct DispatchParams {
  const uint8_t* x;        // [tokens, k]
  const int32_t* ids;      // [tokens, topk]
  int32_t* position;       // [tokens, topk]: read, or (PLAN) written
  int32_t* offsets;        // [experts + 1]: read, or (PLAN) written
  uint8_t* out;            // [tokens * topk, k / 2]
  uint8_t* sf;
  const float* gs;         // [experts]
  int tokens, topk, experts, k;
  int parts;               // CTAs a token
};

constexpr int kDispatchThreads = 128;
constexpr int kMaxTopk = 32;              // a lane of one warp has an assignment each
constexpr int kPlanInDispatch = 512;      // assignments up to which every CTA counts rows for itself

// One CTA per token and 128 blocks.  The token's blocks wait in registers while the warp's lanes fetch where each of its
// assignments goes.  PLAN: the rows are counted here, row = #{j: ids[j] < e} + #{j < i: ids[j] == e}, from all ids in
// shared memory: for a few tokens that is cheaper than a launch of its own (2.3 us).
template <typename Tag, bool V8, bool PLAN>
__global__ void __launch_bounds__(kDispatchThreads) moe_dispatch_kernel(const __grid_constant__ DispatchParams p) {
  __shared__ int all_ids[PLAN ? kPlanInDispatch : 1];
  __shared__ int rows[kMaxTopk], firsts[kMaxTopk];
  const int token = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int nsb = p.k / 16;
  const int col = part * kDispatchThreads + t;
  pdl_wait();
  pdl_launch_dependents();
  uint32_t w[8];
  if (col < nsb) load_block<V8>(p.x + static_cast<int64_t>(token) * p.k * 2 + col * 32, w);
  if constexpr (PLAN) {
    const int n = p.tokens * p.topk;
    for (int j = t; j < n; j += blockDim.x) {
      const int id = __ldg(p.ids + j);
      all_ids[j] = id < 0 || id >= p.experts ? p.experts : id;  // dropped ones sort behind all
    }
    __syncthreads();
    const int warps = blockDim.x >> 5;
    for (int k = warp; k < p.topk; k += warps) {
      const int i = token * p.topk + k, e = all_ids[i];
      int below = 0, before = 0;
      for (int j = lane; j < n; j += 32) {
        below += all_ids[j] < e;
        before += all_ids[j] == e && j < i;
      }
      below = __reduce_add_sync(0xffffffffu, below);
      before = __reduce_add_sync(0xffffffffu, before);
      if (lane == 0) {
        rows[k] = e < p.experts ? below + before : -1;
        firsts[k] = below;
        if (part == 0) p.position[i] = rows[k];
      }
    }
    if (blockIdx.x == 0) {
      __shared__ int start[kMaxGroups + 1];
      for (int e = t; e <= p.experts; e += blockDim.x) start[e] = 0;
      __syncthreads();
      for (int j = t; j < n; j += blockDim.x) atomicAdd(start + all_ids[j], 1);  // integers: no order to matter
      __syncthreads();
      if (warp == 0) scan_experts(start, p.experts, lane);
      __syncthreads();
      for (int e = t; e <= p.experts; e += blockDim.x) p.offsets[e] = start[e];
    }
    __syncthreads();
  }
  // Lane k of every warp has assignment k.
  int row = -1, expert = 0, first = 0;
  float gs = 0.0f;
  if (lane < p.topk) {
    const int64_t i = static_cast<int64_t>(token) * p.topk + lane;
    row = PLAN ? rows[lane] : __ldg(p.position + i);
    if (row >= 0) {
      expert = PLAN ? all_ids[i] : __ldg(p.ids + i);
      first = PLAN ? firsts[lane] : __ldg(p.offsets + expert);
      gs = __ldg(p.gs + expert);
    }
  }
  const int sf_row = ((first >> 7) + expert) * 128 + row - first;
  const float rcp6 = rcp_approx_ftz(6.0f);
  uint32_t sf_byte = 0;
  uint2 packed = make_uint2(0u, 0u);
  float done = 0.0f;
  bool have = false;
  for (int k = 0; k < p.topk; ++k) {
    const int r = __shfl_sync(0xffffffffu, row, k);
    const int sr = __shfl_sync(0xffffffffu, sf_row, k);
    const float scale = __shfl_sync(0xffffffffu, gs, k);
    if (r < 0 || col >= nsb) continue;
    if (!have || scale != done) {
      quantize_block<Tag>(w, scale, rcp_approx_ftz(scale), rcp6, sf_byte, packed);
      done = scale;
      have = true;
    }
    p.sf[sf_offset_128x4(sr, col, nsb)] = static_cast<uint8_t>(sf_byte);
    *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(r) * (p.k >> 1) + col * 8) = packed;
  }
}

template <typename Tag>
int launch_dispatch(const DispatchParams& p, bool v8, bool plan, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.parts) * p.tokens);
  const int threads = p.parts > 1 ? kDispatchThreads : (p.k / 16 + 31) / 32 * 32;
  if (plan)
    return v8 ? launch_dependent(moe_dispatch_kernel<Tag, true, true>, grid, threads, 0, s, p)
              : launch_dependent(moe_dispatch_kernel<Tag, false, true>, grid, threads, 0, s, p);
  return v8 ? launch_dependent(moe_dispatch_kernel<Tag, true, false>, grid, threads, 0, s, p)
            : launch_dependent(moe_dispatch_kernel<Tag, false, false>, grid, threads, 0, s, p);
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

// The histograms of 384 experts exceed the default shared memory; the limit is an attribute per kernel and device.
int allow_histograms(const void* kernel, int which) {
  static std::atomic<bool> configured[2][64] = {};  // setting it twice does no harm
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && configured[which][dev].load(std::memory_order_acquire)) return B2_OK;
  B2_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanWarps * kMaxGroups * 4));
  if (dev >= 0 && dev < 64) configured[which][dev].store(true, std::memory_order_release);
  return B2_OK;
}

// offsets and position of many assignments; `scratch` has a word per assignment (384 counts per 1024 of them fit).
int plan_wide(const int32_t* ids, int32_t* offsets, int32_t* scratch, int32_t* position, int n, int experts, cudaStream_t s) {
  if (int rc = allow_histograms(reinterpret_cast<const void*>(moe_rank_kernel), 1)) return rc;
  const dim3 grid((n + kPlanBlock - 1) / kPlanBlock);
  if (int rc = launch_dependent(moe_count_kernel, grid, dim3(kPlanBlock), 0, s, ids, scratch, n, experts)) return rc;
  return launch_dependent(moe_rank_kernel, grid, dim3(kPlanBlock), static_cast<size_t>(kPlanWarps) * experts * 4, s, ids,
                          static_cast<const int32_t*>(scratch), offsets, position, n, experts);
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
  if (int rc = allow_histograms(reinterpret_cast<const void*>(moe_plan_kernel), 0)) return rc;
  const size_t smem = static_cast<size_t>(kPlanWarps) * experts * 4;
  return launch_dependent(moe_plan_kernel, dim3(1), dim3(kPlanWarps * 32), smem, static_cast<cudaStream_t>(stream), ids_dev,
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

extern "C" int b2_moe_dispatch(const void* x, const int32_t* ids_dev, const float* gs_dev, int32_t* offsets_dev,
                               int32_t* row_token_dev, int32_t* position_dev, void* out, void* sf, int tokens, int topk,
                               int experts, int k, int dtype, void* stream) {
  using namespace b2;
  if (dtype != B2_DTYPE_F16 && dtype != B2_DTYPE_BF16) {
    set_error("b2_moe_dispatch: unsupported dtype %d", dtype);
    return B2_ERR_INVALID_ARGUMENT;
  }
  const int64_t rows = static_cast<int64_t>(tokens) * topk, parts = (static_cast<int64_t>(k) / 16 + kDispatchThreads - 1) / kDispatchThreads;
  if (tokens < 0 || topk < 1 || topk > kMaxTopk || experts < 1 || experts > kMaxGroups || k < 64 || k % 64 != 0 ||
      rows + 128 * (experts + 1) > 0x7fffffffll || parts * tokens > 0x7fffffffll) {
    set_error("b2_moe_dispatch: tokens=%d topk=%d experts=%d k=%d: need tokens >= 0, 1 <= topk <= %d, 1 to %d experts, k %% 64 == 0",
              tokens, topk, experts, k, kMaxTopk, kMaxGroups);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (tokens == 0) return B2_OK;
  if (!x || !ids_dev || !gs_dev || !offsets_dev || !position_dev || !out || !sf || (rows > kPlanInDispatch && !row_token_dev)) {
    set_error("b2_moe_dispatch: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (misaligned(x, 16) || misaligned(out, 8) || misaligned(ids_dev, 4) || misaligned(gs_dev, 4) || misaligned(offsets_dev, 4) ||
      misaligned(row_token_dev, 4) || misaligned(position_dev, 4)) {
    set_error("b2_moe_dispatch: x must be 16-byte, out 8-byte, all else 4-byte aligned");
    return B2_ERR_INVALID_ARGUMENT;
  }
  const bool plan = rows <= kPlanInDispatch;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!plan)
    if (int rc = plan_wide(ids_dev, offsets_dev, row_token_dev, position_dev, tokens * topk, experts, s)) return rc;
  DispatchParams p;
  p.x = static_cast<const uint8_t*>(x);
  p.ids = ids_dev;
  p.position = position_dev;
  p.offsets = offsets_dev;
  p.out = static_cast<uint8_t*>(out);
  p.sf = static_cast<uint8_t*>(sf);
  p.gs = gs_dev;
  p.tokens = tokens;
  p.topk = topk;
  p.experts = experts;
  p.k = k;
  p.parts = static_cast<int>(parts);
  if (dtype == B2_DTYPE_F16) return launch_dispatch<F16Tag>(p, !misaligned(x, 32), plan, s);
  return launch_dispatch<BF16Tag>(p, !misaligned(x, 32), plan, s);
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
  w.y1 = take(inner % 128 ? rows * inner * 4 : 0);  // else the product's epilogue quantizes
  w.a2 = take(rows * (inner / 2));
  w.sf2 = take(tiles * 128 * (inner / 16));
  w.z = take(rows * hidden * 2);
  w.total = at;
  return w;
}
bool ffn_sizes_ok(int tokens, int topk, int experts, int hidden, int inner) {
  return tokens >= 0 && topk >= 1 && topk <= kMaxTopk && experts >= 1 && experts <= kMaxGroups && hidden >= 64 && hidden % 64 == 0 &&
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
    set_error("b2_moe_expert_ffn: tokens=%d topk=%d experts=%d hidden=%d inner=%d: need tokens >= 0, 1 <= topk <= %d, 1 to %d "
              "experts, hidden %% 64 == 0, inner %% 64 == 0", tokens, topk, experts, hidden, inner, kMaxTopk, kMaxGroups);
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
  if (int rc = b2_moe_dispatch(x, ids_dev, gs1_dev, offsets, row_token, position, base + w.a1, base + w.sf1, tokens, topk,
                               experts, hidden, dtype, stream))
    return rc;
  // Both products read early: weights and ids were there before the dispatch, the offsets before the launch in front of
  // the product, but for those that the dispatch itself writes.  There the first product counts the ids.
  const int32_t* counted = rows <= kPlanInDispatch ? ids_dev : nullptr;
  if (inner % 128 == 0) {
    if (int rc = grouped_product_gated(base + w.a1, W1, base + w.sf1, SF1, alpha1_dev, offsets, gs2_dev, base + w.a2,
                                       base + w.sf2, rows, experts, inner, hidden, dtype, true, counted, stream))
      return rc;
  } else {
    if (int rc = grouped_product(base + w.a1, W1, base + w.sf1, SF1, alpha1_dev, offsets, nullptr, base + w.y1, rows, experts,
                                 2 * inner, hidden, dtype, B2_ACT_NONE, true, counted, stream))
      return rc;
    if (int rc = b2_nvfp4_quantize_grouped(base + w.y1, nullptr, offsets, base + w.a2, base + w.sf2, gs2_dev, rows, rows,
                                           experts, inner, dtype, 1, stream))
      return rc;
  }
  if (int rc = grouped_product(base + w.a2, W2, base + w.sf2, SF2, alpha2_dev, offsets, nullptr, base + w.z, rows, experts,
                               hidden, inner, dtype, B2_ACT_NONE, true, nullptr, stream))
    return rc;
  return b2_moe_combine(base + w.z, position, weight_dev, residual, out, rows, tokens, topk, hidden, dtype, stream);
}
