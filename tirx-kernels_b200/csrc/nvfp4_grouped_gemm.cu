// Block-scaled NVFP4 products with a fused epilogue, dense and grouped by expert, for sm_100a:
//
//   D[r, :] = residual[r, :] + act(alpha[g] * A[r, :] B[g]^T + bias[g, :])        for the rows r of group g
//
// A [rows, K] and B [groups, N, K] are E2M1 with one E4M3 scale per 16 values along K; the sum is fp32 in tensor
// memory, everything after it fp32 in registers, with one rounding to the 16-bit output.  The dense product
// (b2_nvfp4_gemm_epilogue) is the grouped one with a single group that has all rows.  Groups are ragged: group g
// has rows offsets[g] .. offsets[g+1] of A and D, read on the device, so a router's result is never waited for by
// the host.  The 128-row tiles of A's scale factors start anew with every group: group g begins at tile
// offsets[g] / 128 + g.  (The next group begins at or behind this one's last tile because
// ceil(n / 128) <= floor((o + n) / 128) - floor(o / 128) + 1; no prefix sum is needed to find a row's scales.)
// B's scale tiles are ceil(N / 128) per group.
//
// The K-slab pipeline is that of nvfp4_gemm.cu: operands by TMA into a ring of stages, scale factors through
// registers into tensor memory, tcgen05.mma by one thread, an epilogue of eight warps.  What differs:
//
//   * the tile list is made on the device: one warp sums the groups' row tiles (a table in shared memory), every
//     role finds (group, row tile, column tile) of its next work item there by bisection;
//   * rows of a tile that belong to the next group are multiplied and dropped: a 32-row part of a tile is stored by
//     the TMA where it lies inside the group, row by row where the group ends inside it;
//   * K needs no multiple of the slab: the TMA fills operands and scales behind K with zeros; columns behind N are
//     multiplied (zeros, or the next group's weights) and dropped;
//   * 32-row tiles for groups of a few rows (AM = 32) may start in any quarter of a 128-row scale tile; the scale
//     warps move that quarter to the first place;
//   * the epilogue runs beside the next tile's products.  Where tensor memory has room for two accumulators (NACC == 2),
//     or a CTA has one tile, it loops over 16 columns of the held one.  The 256 x 256 pair has room for one: 16
//     epilogue warps take it into registers as raw fp32 (64 columns a thread; 8 warps would need 128, hence setmaxnreg)
//     and hand it back before they compute anything; the last tile, which nothing waits for, is held again.
#include <algorithm>
#include <atomic>

#include "nvfp4_tile.cuh"
#include "quant_block.cuh"

namespace b2 {
namespace {

constexpr int kMaxGroups = 384;     // bounds the tables in shared memory
constexpr int kMappedTiles[] = {0, 512, 128};  // per CG: row tiles whose group is looked up; behind them it is searched
constexpr int table_bytes(int cg) { return 2 * (kMaxGroups + 1) * 4 + kMappedTiles[cg] * 2; }
constexpr int kGWarpOperands = 0, kGWarpMma = 1, kGWarpScales = 2, kGWarpMma2 = 3, kGWarpScale0 = 4;

struct GroupedParams {
  const float* alpha;       // [groups]
  const int32_t* offsets;   // [groups + 1], or null: one group with all rows
  const uint16_t* bias;     // [groups, N] or null
  const uint16_t* residual; // [rows, N] or null
  uint16_t* D;              // [rows, N]
  uint32_t* status;
  int rows, groups, N;
  int k_slabs;
  int tiles_m;              // row tiles of the single group when there are no offsets
  int tiles_n, group_n;
  float rcp_tiles_n;        // 1 / tiles_n
  int act;                  // B2_ACT_*
  int fp16;                 // 16-bit type of bias, residual and D
  uint64_t wait_budget_ns;
  // The routed feed-forward's calls (single-CTA tiles): weights and the list of groups were there before the launch in
  // front of this one began, and are read while it runs.
  int early;
  const int32_t* ids;       // [rows] groups of the rows, in any order, to be counted instead of `offsets`, or null
  // kGated: the weight is [gate rows | up rows] of N / 2 each, and SiLU(gate) * up leaves quantized
  const float* gs;          // [groups] encode scale of the output
  uint8_t* out4;            // [rows, N / 4] packed E2M1
  uint8_t* sf_out;          // grouped 128 x 4 scale tiles
};

// What a kernel multiplies and how it ends: one group known to the host; groups; groups, with SiLU(gate) * up quantized.
enum Mode { kDense, kGrouped, kGated };

// A gated tile of a single CTA takes its columns from two places of the weight, half from each: two scale chunks.
template <Mode MODE, int CG, int BN, int STAGES, int TMA_OUT, int AM>
struct GroupedLayout : SmemLayout<CG, BN, STAGES, TMA_OUT, AM, MODE == kGated ? 2 : 0> {
  using Base = SmemLayout<CG, BN, STAGES, TMA_OUT, AM, MODE == kGated ? 2 : 0>;
  static constexpr int kTable = Base::kRingBytes + Base::kBarrierBytes;
  static constexpr int kAll = kTable + (MODE == kDense ? 0 : table_bytes(CG)) + 1024;  // + alignment slack
  static_assert(kAll <= 227 * 1024, "shared memory budget");
};

struct Tile {
  int group, first, last;  // the group and its rows
  int tm, tn;
};

// The groups' row tiles, in shared memory.
struct GroupTable {
  int* starts;       // [groups + 1] row tiles in front of a group
  int* rows;         // [groups + 1] first row of a group
  uint16_t* mapped;  // [mapped_tiles] the group of a row tile
  int mapped_tiles;
};

// Work item t -> its tile.  Every role does this for every tile, the first one in front of its first load: with a
// division in integers, bisection over the groups and the general tile_coords it took 1300 to 1700 cycles, and products
// of little K waited for it (40 groups of one row, N = 4096, K = 512: 22.1 us for 17.7).
template <Mode MODE>
__device__ __forceinline__ Tile find_tile(const GroupedParams& p, const GroupTable& table, int t) {
  Tile r;
  if constexpr (MODE == kDense) {
    r.group = 0;
    r.first = 0;
    r.last = p.rows;
    r.tm = 0;
    r.tn = t;
    if (p.tiles_m > 1) tile_coords(t, p.tiles_m, p.tiles_n, p.group_n, r.tm, r.tn);
    return r;
  }
  int q;
  if (t < (1 << 22)) {  // the product is off by less than one
    q = static_cast<int>(static_cast<float>(t) * p.rcp_tiles_n);
    const int rest = t - q * p.tiles_n;
    q += (rest >= p.tiles_n) - (rest < 0);
  } else {
    q = t / p.tiles_n;
  }
  int lo = 0;
  if (q < table.mapped_tiles) {
    lo = table.mapped[q];
  } else {
    // Among groups without rows, which share a start, bisection ends at the last one, the one that has the tile.
    int hi = p.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (table.starts[mid] <= q) lo = mid;
      else hi = mid;
    }
  }
  r.group = lo;
  r.first = table.rows[lo];
  r.last = table.rows[lo + 1];
  const int before = table.starts[lo], tiles_m = table.starts[lo + 1] - before;
  r.tm = 0;
  r.tn = t - before * p.tiles_n;
  if (tiles_m > 1) tile_coords(r.tn, tiles_m, p.tiles_n, p.group_n, r.tm, r.tn);
  return r;
}

// v / (1 + 2^-(v (c1 + c2 v^2)) ): SiLU with c1 = log2 e, c2 = 0; GELU in its tanh form, since
// (1 + tanh u) / 2 = 1 / (1 + e^-2u), with c1 = 2 log2 e sqrt(2/pi), c2 = 0.044715 c1.  MUFU 2^x and 1/x (relative
// error about 2^-22); 2^-x runs to infinity for very negative v, the quotient to -0.
__device__ __forceinline__ float gate_sigmoid(float v, float c1, float c2) {
  const float e = ex2_approx_ftz(-v * fmaf(c2, v * v, c1));
  return v * rcp_approx_ftz(1.0f + e);
}
// v Phi(v) with the upper tail of the normal distribution by Abramowitz & Stegun 7.1.26 (absolute error 1.5e-7):
// erfc(z) = (a1 t + .. + a5 t^5) e^(-z^2), t = 1 / (1 + p z), z = |v| / sqrt 2.  Two values at once: packed arithmetic, and
// one reciprocal of the product of both denominators (the MUFU is what bounds this step); z is capped where the tail
// has long been zero, so that the product stays finite and one value's infinity or NaN does not reach the other.
__device__ __forceinline__ float2 gelu_erf(float2 v) {
  const float2 z = make_float2(fminf(fabsf(v.x) * 0.70710678118654752f, 64.0f), fminf(fabsf(v.y) * 0.70710678118654752f, 64.0f));
  const float2 d = fma_f32x2(make_float2(0.3275911f, 0.3275911f), z, make_float2(1.0f, 1.0f));
  const float both = rcp_approx_ftz(d.x * d.y);
  const float2 t = mul_f32x2(make_float2(both, both), make_float2(d.y, d.x));
  float2 poly = fma_f32x2(make_float2(1.061405429f, 1.061405429f), t, make_float2(-1.453152027f, -1.453152027f));
  poly = fma_f32x2(poly, t, make_float2(1.421413741f, 1.421413741f));
  poly = fma_f32x2(poly, t, make_float2(-0.284496736f, -0.284496736f));
  poly = fma_f32x2(poly, t, make_float2(0.254829592f, 0.254829592f));
  const float2 w = mul_f32x2(mul_f32x2(z, z), make_float2(-1.4426950408889634f, -1.4426950408889634f));
  const float2 e = make_float2(ex2_approx_ftz(w.x), ex2_approx_ftz(w.y));
  const float2 tail = mul_f32x2(mul_f32x2(poly, t), mul_f32x2(e, make_float2(0.5f, 0.5f)));
  return make_float2(v.x * (v.x >= 0.0f ? 1.0f - tail.x : tail.x), v.y * (v.y >= 0.0f ? 1.0f - tail.y : tail.y));
}

// Not the read-only path: the residual may be the output's own memory (every word is read before it is written, by
// the thread that writes it).
__device__ __forceinline__ uint4 load_residual(const uint16_t* p) {
  uint4 r;
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
// A load whose value nobody uses: what it leaves behind is the line in L1.
__device__ __forceinline__ void touch(const uint16_t* p) {
  asm volatile("{ .reg .b32 a, b, c, d; ld.global.nc.v4.b32 {a, b, c, d}, [%0]; }" ::"l"(p));
}
// 16 columns of a row of the residual, of which `left` (a multiple of 8) are there.
__device__ __forceinline__ void load_next(const uint16_t* p, int left, uint4 (&r)[2]) {
  if (left > 0) r[0] = load_residual(p);
  if (left > 8) r[1] = load_residual(p + 8);
}

// ---- the epilogue's steps, each over all of a warp's columns of one row, in place --------------------------------------
// One step after another, with the choice of activation or type outside the loop: what a call does not use it does not
// fetch.  With the choices inside, eight columns at a time, the instructions that a short launch jumped over cost it
// 1 to 2 us (16 x 8192 x 8192 11.4 us for 10.6).
template <typename Tag, int COLS>
__device__ __forceinline__ void add_bias(const uint16_t* bias, int left, uint32_t* v) {
#pragma unroll
  for (int c = 0; c < COLS / 8; ++c) {
    if (8 * c < left) {
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(bias + 8 * c));
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[8 * c + 2 * i] = __float_as_uint(__uint_as_float(v[8 * c + 2 * i]) + unpack_lo<Tag>(w[i]));
        v[8 * c + 2 * i + 1] = __float_as_uint(__uint_as_float(v[8 * c + 2 * i + 1]) + unpack_hi<Tag>(w[i]));
      }
    }
  }
}
template <int COLS>
__device__ __forceinline__ void activate(int act, uint32_t* v) {
  if (act == B2_ACT_SILU || act == B2_ACT_GELU_TANH) {
    const float c1 = act == B2_ACT_SILU ? 1.4426950408889634f : 2.3022081983375f;
    const float c2 = act == B2_ACT_SILU ? 0.0f : 0.10294324f;
#pragma unroll
    for (int i = 0; i < COLS; ++i) v[i] = __float_as_uint(gate_sigmoid(__uint_as_float(v[i]), c1, c2));
  } else if (act == B2_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < COLS; i += 2) {
      const float2 g = gelu_erf(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
      v[i] = __float_as_uint(g.x);
      v[i + 1] = __float_as_uint(g.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < COLS; ++i) v[i] = __uint_as_float(v[i]) < 0.0f ? 0u : v[i];  // ReLU; a NaN stays one
  }
}
template <typename Tag>
__device__ __forceinline__ void add8(uint4 r, uint32_t* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __float_as_uint(__uint_as_float(v[2 * i]) + unpack_lo<Tag>(w[i]));
    v[2 * i + 1] = __float_as_uint(__uint_as_float(v[2 * i + 1]) + unpack_hi<Tag>(w[i]));
  }
}
// The one rounding: words 0 .. N/2 - 1 become the packed columns.
template <typename Tag, int N>
__device__ __forceinline__ void pack(uint32_t* v) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) v[i] = pack_pair<Tag>(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])));
}

__device__ __forceinline__ void lds64(uint32_t addr, uint32_t* r) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
}
__device__ __forceinline__ uint4 lds128_vec(uint32_t addr) {
  uint32_t r[4];
  lds128(addr, r);
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// Asks L2 for a box of a tensor map.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
template <int REGS>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}

// 16 gate and 16 up columns of one row -> a block of SiLU(gate) * up in NVFP4, with the bits that the 16-bit product
// followed by the quantizer's fuse_silu gives (the same roundings: product to 16 bits, SiLU * up to 16 bits).
// WIDE: four pairs' chains side by side (8 rows of 8 groups, 2048 x 4096, 10.8 -> 10.1 us); where the registers hold a whole
// tile, that spills (8192 rows of 8, 4096 x 4096: 61.7 -> 62.8), and one pair follows the other.
template <typename Tag, bool WIDE>
__device__ __forceinline__ void gated_block(const uint32_t* gate, const uint32_t* up, float alpha, float gs, uint32_t& sf_byte,
                                            uint2& packed) {
  uint32_t w[8];
  auto scaled = [&](const uint32_t* v, int i) {
    return pack_pair<Tag>(make_float2(__uint_as_float(v[2 * i]) * alpha, __uint_as_float(v[2 * i + 1]) * alpha));
  };
  if constexpr (WIDE) {
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      const uint32_t g[4] = {scaled(gate, h), scaled(gate, h + 1), scaled(gate, h + 2), scaled(gate, h + 3)};
      const uint32_t u[4] = {scaled(up, h), scaled(up, h + 1), scaled(up, h + 2), scaled(up, h + 3)};
      uint32_t o[4];
      silu_and_mul_4<Tag>(g, u, o);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[h + i] = o[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = silu_and_mul_pair<Tag>(scaled(gate, i), scaled(up, i));
  }
  quantize_block<Tag>(w, gs, rcp_approx_ftz(gs), rcp_approx_ftz(6.0f), sf_byte, packed);
}
// Where a row's scale of column `col` (a multiple of 16) lies, `inner` columns a row.
__device__ __forceinline__ int64_t gated_sf_offset(int64_t sf_row, int col, int inner) {
  return (col / 16 & 3) + static_cast<int64_t>(col / 64) * 512 + (sf_row & 31) * 16 + ((sf_row & 127) >> 5) * 4 +
         (sf_row >> 7) * (8 * static_cast<int64_t>(inner));
}

// CG: CTAs of a tile (1 or 2).  BN: its columns.  AM: rows of A that one CTA loads and multiplies (the MMA reads 128;
// what follows a shorter box in the stage only reaches accumulator rows that nobody reads).  MMAS: MMA-issuing warps
// with an accumulator each, for a single tile per CTA (issuing is the limit there).  NACC: accumulators in turn, for many tiles.
// SETS of 4 scale warps and PARTS of 4 epilogue warps, each with BN / PARTS columns.
constexpr int group_threads(int sets, int parts) { return 32 * (4 + 4 * sets + 4 * parts); }
// Registers a thread of each warpgroup has when PARTS == 4 (768 threads start with 80 each): 6 x 80 = 56 + 40 + 4 x 96.
constexpr int kRegsLaunch = 80, kRegsIssue = 56, kRegsScale = 40, kRegsEpilogue = 96;
static_assert(kRegsIssue + kRegsScale + 4 * kRegsEpilogue <= 6 * kRegsLaunch, "no warpgroup waits for registers that nobody gives");

template <Mode MODE, int CG, int BN, int STAGES, int TMA_OUT, int AM, int MMAS, int NACC, int SETS, int PARTS>
__global__ void __launch_bounds__(group_threads(SETS, PARTS), 1)
    nvfp4_grouped_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                              const __grid_constant__ CUtensorMap map_sfa, const __grid_constant__ CUtensorMap map_sfb,
                              const __grid_constant__ CUtensorMap map_d, const __grid_constant__ CUtensorMap map_r,
                              const __grid_constant__ GroupedParams p) {
  using L = GroupedLayout<MODE, CG, BN, STAGES, TMA_OUT, AM>;
  static_assert(MMAS == 1 || (CG == 1 && TMA_OUT == 0), "the second MMA warp exists for single-CTA tiles");
  static_assert(CG == 1 || AM == kBlockM, "pairs load all rows");
  // A stage's slabs belong to one issuer then.  With an odd ring the other issuer may still wait for the stage's last slab
  // when this one polls for the next: the parity of the phase in front of that slab's is the one it asks for, and it would
  // take the poll for its own slab's.
  static_assert(STAGES % MMAS == 0, "two issuers need an even ring");
  constexpr int kBM = AM * CG;                // rows of a tile
  constexpr int kAccCols = BN * MMAS * NACC;  // accumulator columns in front of the stages' scale areas
  static_assert(kAccCols + STAGES * L::kSfCols <= 512, "tensor memory budget");
  constexpr int kTmemCols = 512;
  constexpr uint32_t kIdesc = instr_desc(kBlockM * CG, BN);
  constexpr uint32_t kOperandTx = static_cast<uint32_t>(L::kABytes + L::kBBytes) * CG;
  constexpr uint32_t kScaleTx = static_cast<uint32_t>(L::kSfaBytes + L::kSfbBytes);
  constexpr bool kWarpWide = CG == 2;  // issuing roles run as whole warps (see nvfp4_gemm.cu)
  constexpr int kCols = BN / PARTS;    // columns of an epilogue warp
  constexpr int kOuts = kCols / 2;     // gated: its outputs
  constexpr int kWarpEpi0 = kGWarpScale0 + 4 * SETS;
  constexpr bool kMoveRegisters = PARTS == 4;
  static_assert((kCols == 32 || kCols == 64) && (!kMoveRegisters || SETS == 1), "epilogue shapes");

  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + L::kRingBytes;
  // The barriers of nvfp4_gemm.cu: full (operands landed and scales in tensor memory, on the pair's leader), sfload
  // (scale blocks landed in shared memory), empty (the stage's MMAs retired); per accumulator full and empty.
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto sfload_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto empty_bar = [&](int s) { return bar_base + 8u * (2 * STAGES + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (3 * STAGES + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (3 * STAGES + NACC + a); };
  constexpr int kResBarOffset = (3 * STAGES + 2 * NACC) * 8 + 16;  // residual landed, per epilogue warp
  static_assert(kResBarOffset + 32 * PARTS <= L::kBarrierBytes, "barrier area");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + L::kRingBytes + 8 * (3 * STAGES + 2 * NACC));
  volatile uint32_t* abort_flag = tmem_slot + 1;
  int* starts = reinterpret_cast<int*>(smem_gen + L::kTable);
  const GroupTable table{starts, starts + kMaxGroups + 1, reinterpret_cast<uint16_t*>(starts + 2 * (kMaxGroups + 1)),
                         kMappedTiles[CG]};
  const WaitCtx ctx{p.status, abort_flag, p.wait_budget_ns};

  const int warp = kWarpWide ? __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0)
                             : static_cast<int>(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? __shfl_sync(0xffffffffu, cluster_ctarank(), 0) : 0u;
  const bool leader = rank == 0;
  const int unit = CG == 2 ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int num_units = CG == 2 ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1 + 4 * CG);  // the producer's expect_tx arrive + one arrive per scale warp of the group
      mbar_init(sfload_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < NACC; ++a) {
      mbar_init(acc_full_bar(a), MMAS);
      mbar_init(acc_empty_bar(a), 4 * PARTS * CG);  // one arrive per epilogue warp of every CTA in the group
    }
    if constexpr (TMA_OUT > 0)
      for (int w = 0; w < 4 * PARTS; ++w) mbar_init(bar_base + kResBarOffset + 8u * w, 1);
    *abort_flag = 0u;
    fence_barrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
    prefetch_tmap(&map_sfa);
    prefetch_tmap(&map_sfb);
  }
  if (warp == kGWarpMma) {
    tmem_alloc<CG>(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish<CG>();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = kWarpWide ? __shfl_sync(0xffffffffu, *tmem_slot, 0) : *tmem_slot;
  // Dependent launch as in nvfp4_gemm.cu: nothing in front of this wait touches global memory.  The exception are early
  // calls.  Their predecessor let them start behind its own wait, so everything in front of it is complete: the table of
  // groups and the first weights are read beside it (one token through 8 experts of 64,
  // 4096 x 1024: 28.3 us for 29.9).
  constexpr bool kMayBeEarly = CG == 1 && MODE != kDense;
  const bool early = kMayBeEarly && p.early;
  auto dependent_launch = [] {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  };
  if (!early) dependent_launch();
  if constexpr (MODE != kDense) {
    if (warp == kGWarpMma2) {
      const bool counted = kMayBeEarly && p.ids;
      if (counted) {
        for (int g = lane; g < p.groups; g += 32) starts[g] = 0;
        __syncwarp();
#pragma unroll 4
        for (int i = lane; i < p.rows; i += 32) {
          const int id = __ldcg(p.ids + i);
          if (id >= 0 && id < p.groups) atomicAdd(starts + id, 1);
        }
        __syncwarp();
      }
      int tiles = 0, rows = 0;  // row tiles, counted rows in front of the 32 groups of this step
      for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        int first = 0, last = 0;
        if (counted) {
          const int count = g < p.groups ? starts[g] : 0;
          last = count;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, last, d);
            if (lane >= d) last += up;
          }
          last += rows;
          first = last - count;
          rows = __shfl_sync(0xffffffffu, last, 31);
        } else if (g < p.groups) {
          // Offsets that are not ascending or leave [0, rows] are brought back into it: no access leaves A or D.
          first = min(max(__ldcg(p.offsets + g), 0), p.rows);
          last = min(max(__ldcg(p.offsets + g + 1), first), p.rows);
        }
        const int mine = (last - first + kBM - 1) / kBM;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, d);
          if (lane >= d) sum += up;
        }
        if (g < p.groups) {
          const int start = tiles + sum - mine;
          starts[g] = start;
          table.rows[g] = first;
          if (g == p.groups - 1) {
            starts[g + 1] = tiles + sum;
            table.rows[g + 1] = last;
          }
          for (int q = start; q < start + mine && q < table.mapped_tiles; ++q) table.mapped[q] = static_cast<uint16_t>(g);
        }
        tiles += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    __syncthreads();
  }
  if (early && warp != kGWarpOperands && warp != kGWarpScales) dependent_launch();
  // What the issuing warps compute from shared memory is made uniform by a shuffle, or the compiler would keep their
  // loops' state out of uniform registers (nvfp4_gemm.cu).
  auto uniform = [](int v) { return kWarpWide ? __shfl_sync(0xffffffffu, v, 0) : v; };
  const int num_tiles = MODE != kDense ? uniform(starts[p.groups]) * p.tiles_n : p.tiles_m * p.tiles_n;
  const int k_slabs = p.k_slabs;

  // The waits of the issuing roles: of the whole warp with one outcome, or of lane 0.
  auto role_wait = [&](uint32_t bar, uint32_t phase, uint32_t code) {
    const bool ok = wait_or_abort(bar, phase, ctx, code);
    if constexpr (kWarpWide) return __all_sync(0xffffffffu, ok) != 0;
    else return ok;
  };
  // The epilogue's waits: one outcome for all lanes, since the warp goes on with __syncwarp.  (The scale warps poll
  // converged as in nvfp4_gemm.cu: the vote would cost them 4 % of a decode product, once per slab.)
  auto warp_wait = [&](uint32_t bar, uint32_t phase, uint32_t code) {
    return __all_sync(0xffffffffu, wait_or_abort(bar, phase, ctx, code)) != 0;
  };
  auto issues = [&] { return kWarpWide ? elect_one() : true; };

  // setmaxnreg stands in front of the roles of its warpgroup, inside one branch: behind a point where branches with
  // different limits meet, the compiler keeps to the lowest.
  if (warp < kGWarpScale0) {
    if constexpr (kMoveRegisters) give_registers<kRegsIssue>();
    if (warp == kGWarpOperands) {
      // ================= TMA producer of the operands =================
      if (kWarpWide || lane == 0) {
        // Gated: the first half of the tile's columns are gates, the second (the pair's second CTA's) the matching ups.
        auto first_row_b = [&](const Tile& tile) {
          return MODE == kGated ? uniform(tile.group * p.N + tile.tn * (BN / 2)) + static_cast<int>(rank) * (p.N / 2)
                                : uniform(tile.group * p.N + tile.tn * BN) + static_cast<int>(rank) * L::kBRows;
        };
        auto load_b = [&](uint32_t sbase, int ks, int row_b, uint32_t op_bar) {
          tma_load_2d<CG>(sbase + L::kABytes, &map_b, ks * 128, row_b, op_bar);
          if constexpr (MODE == kGated && CG == 1)
            tma_load_2d<CG>(sbase + L::kABytes + L::kBBytes / 2, &map_b, ks * 128, row_b + p.N / 2, op_bar);
        };
        int ahead = 0;  // slabs whose B is on its way
        if constexpr (kMayBeEarly) {
          if (early) {
            for (int t = unit; t < num_tiles && ahead < STAGES; t += num_units) {
              const int row_b = first_row_b(find_tile<MODE>(p, table, t));
              for (int ks = 0; ks < k_slabs && ahead < STAGES; ++ks, ++ahead) {
                mbar_expect_tx(full_bar(ahead), kOperandTx);
                load_b(smem_base + ahead * L::kStageBytes, ks, row_b, full_bar(ahead));
              }
            }
            dependent_launch();
          }
        }
        int stage = 0;
        uint32_t phase = 0;
        bool alive = true;
        for (int t = unit; t < num_tiles && alive; t += num_units) {
          const Tile tile = find_tile<MODE>(p, table, t);
          const int row_a = uniform(tile.first + tile.tm * kBM) + static_cast<int>(rank) * kBlockM;
          const int row_b = first_row_b(tile);
          for (int ks = 0; ks < k_slabs; ++ks) {
            if (!role_wait(empty_bar(stage), phase ^ 1u, 1u)) { alive = false; break; }
            const uint32_t sbase = smem_base + stage * L::kStageBytes;
            // operand bytes of both CTAs of a pair are counted on the leader's barrier
            const uint32_t op_bar = CG == 2 ? mapa_shared(full_bar(stage), 0) : full_bar(stage);
            if (issues()) {
              if (kMayBeEarly && ahead > 0) {
                --ahead;
                tma_load_2d<CG>(sbase, &map_a, ks * 128, row_a, op_bar);
              } else {
                if (leader) mbar_expect_tx(full_bar(stage), kOperandTx);
                tma_load_2d<CG>(sbase, &map_a, ks * 128, row_a, op_bar);
                load_b(sbase, ks, row_b, op_bar);
              }
            }
            if constexpr (kWarpWide) __syncwarp();
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          }
        }
      }
    } else if (warp == kGWarpScales) {
      // ================= TMA producer of the scale factors =================
      if (kWarpWide || lane == 0) {
        const int sfb_tiles = (p.N + 127) / 128;
        auto first_tile_b = [&](const Tile& tile) {
          return uniform(tile.group * sfb_tiles + (tile.tn * (MODE == kGated ? BN / 2 : BN)) / 128);
        };
        auto load_b = [&](uint32_t sf_smem, int ks, int sfb_tile, uint32_t bar) {
          tma_load_3d<1>(sf_smem + L::kSfaBytes, &map_sfb, 0, ks * 4, sfb_tile, bar);
          if constexpr (MODE == kGated)
            tma_load_3d<1>(sf_smem + L::kSfaBytes + 2048, &map_sfb, 0, ks * 4, sfb_tile + p.N / 256, bar);
        };
        int ahead = 0;  // slabs whose scales of B are on their way
        if constexpr (kMayBeEarly) {
          if (early) {
            for (int t = unit; t < num_tiles && ahead < STAGES; t += num_units) {
              const int sfb_tile = first_tile_b(find_tile<MODE>(p, table, t));
              for (int ks = 0; ks < k_slabs && ahead < STAGES; ++ks, ++ahead) {
                mbar_expect_tx(sfload_bar(ahead), kScaleTx);
                load_b(smem_base + ahead * L::kStageBytes + L::kABytes + L::kBBytes, ks, sfb_tile, sfload_bar(ahead));
              }
            }
            dependent_launch();
          }
        }
        int stage = 0;
        uint32_t phase = 0;
        bool alive = true;
        for (int t = unit; t < num_tiles && alive; t += num_units) {
          const Tile tile = find_tile<MODE>(p, table, t);
          const int sfa_tile = uniform((tile.first >> 7) + tile.group + ((tile.tm * kBM) >> 7)) + static_cast<int>(rank);
          const int sfb_tile = first_tile_b(tile);
          for (int ks = 0; ks < k_slabs; ++ks) {
            if (!role_wait(empty_bar(stage), phase ^ 1u, 1u)) { alive = false; break; }
            const uint32_t sf_smem = smem_base + stage * L::kStageBytes + L::kABytes + L::kBBytes;
            if (issues()) {
              if (kMayBeEarly && ahead > 0) {
                --ahead;
                tma_load_3d<1>(sf_smem, &map_sfa, 0, ks * 4, sfa_tile, sfload_bar(stage));
              } else {
                mbar_expect_tx(sfload_bar(stage), kScaleTx);
                tma_load_3d<1>(sf_smem, &map_sfa, 0, ks * 4, sfa_tile, sfload_bar(stage));
                load_b(sf_smem, ks, sfb_tile, sfload_bar(stage));
              }
            }
            if constexpr (kWarpWide) __syncwarp();
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          }
        }
      }
    } else if (warp == kGWarpMma || (MMAS == 2 && warp == kGWarpMma2)) {
      // ================= MMA issuer(s), in the leader =================
      // Issuer `me` takes the K slabs with index % MMAS == me and adds them up in its own columns.
      const int me = warp == kGWarpMma ? 0 : 1;
      if (leader && (kWarpWide || lane == 0)) {
        bool alive = true;
        int acc = 0;
        uint32_t acc_phase = 0;
        int slab0 = 0;  // slabs of the tiles that are done: the ring position of this tile's first slab
        for (int t = unit; t < num_tiles && alive; t += num_units, slab0 += k_slabs) {
          if (!role_wait(acc_empty_bar(acc), acc_phase ^ 1u, 2u)) break;
          tc_fence_after();
          // A 64-wide tile uses half of a 128-row scale chunk of B: the upper half starts two columns in.
          uint32_t sfb_half = 0;
          if constexpr (BN == 64) sfb_half = static_cast<uint32_t>(find_tile<MODE>(p, table, t).tn & 1) * 2u;
          const uint32_t acc_tmem = tmem_base + static_cast<uint32_t>((acc * MMAS + me) * BN);
          int stage = (slab0 + me) % STAGES;
          uint32_t phase = static_cast<uint32_t>((slab0 + me) / STAGES) & 1u;
          bool polled = false;  // the poll issued with the previous slab found this slab's barrier complete
          for (int ks = me; ks < k_slabs; ks += MMAS) {
            if (!polled && !role_wait(full_bar(stage), phase, 3u)) { alive = false; break; }
            tc_fence_after();
            const uint32_t sbase = smem_base + stage * L::kStageBytes;
            const uint32_t sf_tmem = tmem_base + kAccCols + stage * L::kSfCols;
            const uint64_t a_desc = operand_desc(sbase), b_desc = operand_desc(sbase + L::kABytes);
            int next_stage = stage + MMAS;
            uint32_t next_phase = phase;
            if (next_stage >= STAGES) { next_stage -= STAGES; next_phase ^= 1u; }
            if constexpr (kWarpWide) {
              if (elect_one()) {
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
                  tc_mma<CG>(acc_tmem, a_desc + 2 * kb, b_desc + 2 * kb, kIdesc, sf_tmem + kb * 4,
                             sf_tmem + 16 + kb * 4 * L::kChunks + sfb_half, (ks >= MMAS || kb) ? 1u : 0u);
                tc_commit_pair(empty_bar(stage));
              }
              __syncwarp();
            } else {
              const bool more = ks + MMAS < k_slabs;  // behind the last slab the poll asks this slab's own barrier
              const uint32_t ok = tc_slab_and_poll_next<CG>(
                  acc_tmem, a_desc, b_desc, kIdesc, sf_tmem, sf_tmem + 16 + sfb_half, 4 * L::kChunks,
                  ks >= MMAS ? 1u : 0u, empty_bar(stage), full_bar(more ? next_stage : stage),
                  more ? next_phase : phase);
              polled = more && ok != 0;
            }
            stage = next_stage;
            phase = next_phase;
          }
          if (!alive) break;
          if (issues()) {
            if constexpr (CG == 2) tc_commit_pair(acc_full_bar(acc));
            else tc_commit<CG>(acc_full_bar(acc));
          }
          if constexpr (kWarpWide) __syncwarp();
          if (++acc == NACC) { acc = 0; acc_phase ^= 1u; }
        }
      }
    }
  } else if (warp < kWarpEpi0) {
    if constexpr (kMoveRegisters) give_registers<kRegsScale>();
    // ================= scale warps: shared memory -> registers -> tensor memory =================
    // Layout and reasons as in nvfp4_gemm.cu.  Two sets of four warps share the stages by parity; one set is enough
    // where a slab's products take longer (256 columns: 520 cycles) than the way of its scales (about 250).
    const int quarter = warp & 3;
    const int set = (warp - kGWarpScale0) >> 2;
    const int total_slabs = unit < num_tiles ? ((num_tiles - unit + num_units - 1) / num_units) * k_slabs : 0;
    constexpr bool kHalves = MODE == kGated && CG == 1;  // 64 gate and 64 up columns, each half of a scale chunk
    int tile_slabs = 0, t = unit;  // slabs left of the current tile, the next tile (AM == 32 and kHalves only)
    int part = 0;                  // the 32-row quarter of the scale tile that this tile's rows have
    uint32_t half_bytes = 0;       // the 64-row half of the scale chunks that this tile's columns have
    for (int n = 0; n < total_slabs; ++n) {
      if constexpr (AM == 32 || kHalves) {
        if (tile_slabs == 0) {
          const Tile tile = find_tile<MODE>(p, table, t);
          part = tile.tm & 3;
          half_bytes = static_cast<uint32_t>(tile.tn & 1) * 8u;
          t += num_units;
          tile_slabs = k_slabs;
        }
        --tile_slabs;
      }
      const int stage = n % STAGES;
      if (SETS == 2 && (stage & 1) != set) continue;
      const uint32_t phase = static_cast<uint32_t>(n / STAGES) & 1u;
      if (!wait_or_abort(sfload_bar(stage), phase, ctx, 5u)) break;
      const uint32_t sfa_smem = smem_base + stage * L::kStageBytes + L::kABytes + L::kBBytes + lane * 16;
      const uint32_t sfb_smem = sfa_smem + L::kSfaBytes;
      const uint32_t dst = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + kAccCols + stage * L::kSfCols;
      // The whole slab's words at once, or, where the epilogue wants the registers, sixteen at a time.
      auto load_b = [&](int c, uint32_t* b) {  // words 16 c .. 16 c + 15 of [kb][chunk][4]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kHalves) {  // [kb][gate 2, up 2]
            lds64(sfb_smem + i * 512 + half_bytes, b + 4 * i);
            lds64(sfb_smem + 2048 + i * 512 + half_bytes, b + 4 * i + 2);
            continue;
          }
          const int word = 4 * c + i;
          lds128(sfb_smem + ((word % L::kChunks) * 4 + word / L::kChunks) * 512, b + 4 * i);
        }
      };
      uint32_t a[16], ahead[kMoveRegisters ? 1 : 16 * L::kChunks];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) lds128(sfa_smem + kb * 512, a + 4 * kb);
      if constexpr (!kMoveRegisters) {
#pragma unroll
        for (int c = 0; c < L::kChunks; ++c) load_b(c, ahead + 16 * c);
      }
      if constexpr (AM == 32) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const uint32_t low = part & 1 ? a[4 * kb + 1] : a[4 * kb], high = part & 1 ? a[4 * kb + 3] : a[4 * kb + 2];
          a[4 * kb] = part & 2 ? high : low;
        }
      }
      tmem_st_32x32_x16(dst, a);
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) {
        if constexpr (kMoveRegisters) {
          uint32_t b[16];
          load_b(c, b);
          tmem_st_32x32_x16(dst + 16 + 16 * c, b);
        } else {
          tmem_st_32x32_x16(dst + 16 + 16 * c, ahead + 16 * c);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive_local(full_bar(stage));
        else mbar_arrive_cluster_relaxed(mapa_shared(full_bar(stage), 0));
      }
    }
  } else {
    if constexpr (kMoveRegisters) take_registers<kRegsEpilogue>();
    // ================= epilogue: lane quarter = warp & 3, column part = (warp - first) / 4 ===========
    constexpr bool kAlwaysHold = NACC == 2 || MMAS == 2;  // see hold_tile
    const int quarter = warp & 3;
    const int part = (warp - kWarpEpi0) >> 2;
    const uint64_t store_policy = l2_policy_evict_first();
    const bool two = MMAS == 2 && k_slabs > 1;  // a single slab leaves the second issuer without one
    // Staging of the TMA store: buffers of 16 rows x 64 columns per warp, 128-byte rows, 128-byte swizzle.  (Boxes of
    // 32 x 32, with 64-byte rows, take the TMA twice as long: 16384 rows of 32 groups, N = 2048, K = 1408: 98 us for 49.)
    static_assert(TMA_OUT == 0 || kCols == 64, "store boxes");
    constexpr int kBufs = TMA_OUT > 0 ? L::kStagingBytes / (4 * PARTS * 2048) : 1;
    static_assert(kBufs == 1 || kBufs == 2, "store buffers");
    const uint32_t staging = smem_base + STAGES * L::kStageBytes + static_cast<uint32_t>(warp - kWarpEpi0) * kBufs * 2048u;
    const uint32_t res_bar = bar_base + kResBarOffset + 8u * static_cast<uint32_t>(warp - kWarpEpi0);
    uint32_t res_phase = 0;
    int acc = 0;
    uint32_t acc_phase = 0;

    // This warp's part of a tile.
    struct Part {
      Tile tile;
      float alpha;
      int row0, row, col0;
      bool any, mine;         // the warp has rows and columns here; the lane has a row
      int64_t at;             // of the lane's first element in D
      const uint16_t* bias;   // of the warp's first column, or null
    };
    auto part_of = [&](int t) {
      Part w;
      w.tile = find_tile<MODE>(p, table, t);
      w.alpha = __ldg(p.alpha + w.tile.group);
      const int in_tile = static_cast<int>(rank) * kBlockM + quarter * 32;
      w.row0 = w.tile.first + w.tile.tm * kBM + in_tile;
      w.row = w.row0 + lane;
      w.col0 = w.tile.tn * BN + part * kCols;
      w.any = in_tile < kBM && w.row0 < w.tile.last && (MODE == kGated || w.col0 < p.N);
      w.mine = w.any && w.row < w.tile.last;
      w.at = static_cast<int64_t>(w.row) * p.N + w.col0;
      w.bias = p.bias ? p.bias + static_cast<int64_t>(w.tile.group) * p.N + w.col0 : nullptr;
      if (w.bias && w.any && lane < kCols / 8 && w.col0 + 8 * lane < p.N) touch(w.bias + 8 * lane);  // into L1
      return w;
    };
    // The TMA clips rows behind the last row and columns behind N, but knows nothing of groups.
    auto whole = [&](const Part& w) { return TMA_OUT > 0 && (w.row0 + 32 <= w.tile.last || w.tile.last == p.rows); };
    auto give_back = [&] {  // the accumulator
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive_local(acc_empty_bar(acc));
        else mbar_arrive_cluster_relaxed(mapa_shared(acc_empty_bar(acc), 0));
      }
      if (++acc == NACC) { acc = 0; acc_phase ^= 1u; }
    };
    auto sf_row_of = [&](const Part& w) {
      return (static_cast<int64_t>(w.tile.first >> 7) + w.tile.group) * 128 + w.row - w.tile.first;
    };

    // A tile that stays in tensor memory while the epilogue loops over 16 columns at a time: nothing waits for the
    // accumulator (there is another, or no further tile), and few registers are needed: the rolled loop took grouped
    // products of one wave from 9.7 to 8.5 us (777 rows of 7, N = 1352, K = 1088), decode ones from 40 to 38.  (32 columns
    // at a time: 200 x 4096 x 4096 7.1 us for 6.4, 256 x 8192 x 8192 11.6 for 10.9.)
    auto hold_tile = [&](int t) {
      const Part w = part_of(t);
      // All 32 rows at once: in the warp's two buffers, or, where it has one, in the ring, whose last products are done
      // when this tile's accumulator is (row-strided stores of a last tile took 4 us for 1).
      const bool staged = whole(w);
      const bool res_staged = staged && p.residual;
      const uint32_t buffers = kBufs == 2 ? staging : smem_base + static_cast<uint32_t>(warp - kWarpEpi0) * 4096u;
      static_assert(TMA_OUT == 0 || kBufs == 2 || 4 * PARTS * 4096 <= STAGES * L::kStageBytes, "buffers in the ring");
      auto request_residual = [&] {
        if constexpr (TMA_OUT > 0) {
          mbar_expect_tx(res_bar, 4096u);
          tma_load_2d<1>(buffers, &map_r, w.col0, w.row0, res_bar);
          tma_load_2d<1>(buffers + 2048u, &map_r, w.col0, w.row0 + 16, res_bar);
        }
      };
      if constexpr (TMA_OUT > 0) {
        if (res_staged && w.any && lane == 0) {
          if (kBufs == 2) {
            bulk_wait_read<0>();  // the stores of the last tile have read the buffers
            request_residual();
          } else {
            tma_prefetch_2d(&map_r, w.col0, w.row0);
            tma_prefetch_2d(&map_r, w.col0, w.row0 + 16);
          }
        }
      }
      const uint16_t* direct = p.residual && !res_staged && w.mine ? p.residual + w.at : nullptr;
      uint4 next[2];  // the residual's 16 columns of the next step
      if (direct) load_next(direct, p.N - w.col0, next);
      if (!warp_wait(acc_full_bar(acc), acc_phase, 4u)) return false;
      tc_fence_after();
      if (w.any) {
        if (TMA_OUT > 0 && staged) {
          if (res_staged) {
            if (kBufs == 1 && lane == 0) request_residual();
            if (!warp_wait(res_bar, res_phase, 6u)) return false;
            res_phase ^= 1u;
          } else {
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
          }
        }
        const uint32_t acc_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * MMAS * BN);
        const uint32_t here = buffers + static_cast<uint32_t>(lane >> 4) * 2048u + (lane & 15) * 128u;
        const float gs = MODE == kGated ? __ldg(p.gs + w.tile.group) : 0.0f;
#pragma unroll 1
        for (int c0 = 0; c0 < (MODE == kGated ? kOuts : kCols); c0 += 16) {
          uint32_t v[16];
          if constexpr (MODE == kGated) {
            uint32_t up[16];
            tmem_ld_32x16(acc_tmem + part * kOuts + c0, v);
            tmem_ld_32x16(acc_tmem + BN / 2 + part * kOuts + c0, up);
            tmem_ld_wait();
            if (w.mine) {
              const int col = w.tile.tn * (BN / 2) + part * kOuts + c0;
              uint32_t sf_byte;
              uint2 packed;
              if (p.fp16) gated_block<F16Tag, true>(v, up, w.alpha, gs, sf_byte, packed);
              else gated_block<BF16Tag, true>(v, up, w.alpha, gs, sf_byte, packed);
              p.sf_out[gated_sf_offset(sf_row_of(w), col, p.N / 2)] = static_cast<uint8_t>(sf_byte);
              *reinterpret_cast<uint2*>(p.out4 + static_cast<int64_t>(w.row) * (p.N / 4) + col / 2) = packed;
            }
            continue;
          }
          tmem_ld_32x16(acc_tmem + part * kCols + c0, v);
          if (MMAS == 2 && two) {
            uint32_t second[16];
            tmem_ld_32x16(acc_tmem + BN + part * kCols + c0, second);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(second[i]));
          } else {
            tmem_ld_wait();
          }
          const int left = p.N - w.col0 - c0;
          if (left <= 0) break;  // the same in the whole warp
          uint4 r[2] = {next[0], next[1]};
          if (direct && c0 + 16 < kCols) load_next(direct + c0 + 16, left - 16, next);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * w.alpha);
          if (w.bias) {
            if (p.fp16) add_bias<F16Tag, 16>(w.bias + c0, left, v);
            else add_bias<BF16Tag, 16>(w.bias + c0, left, v);
          }
          if (p.act != B2_ACT_NONE) activate<16>(p.act, v);
          const uint32_t at0 = here + (((static_cast<uint32_t>(c0) >> 3) ^ (lane & 7u)) * 16u);
          const uint32_t at1 = here + ((((static_cast<uint32_t>(c0) >> 3) + 1u) ^ (lane & 7u)) * 16u);
          if (TMA_OUT > 0 && res_staged) {
            r[0] = lds128_vec(at0);
            r[1] = lds128_vec(at1);
          }
          if (p.residual) {  // lanes without a row add whatever lies in r and store nothing
            if (p.fp16) {
              add8<F16Tag>(r[0], v);
              add8<F16Tag>(r[1], v + 8);
            } else {
              add8<BF16Tag>(r[0], v);
              add8<BF16Tag>(r[1], v + 8);
            }
          }
          if (p.fp16) pack<F16Tag, 16>(v);
          else pack<BF16Tag, 16>(v);
          if (TMA_OUT > 0 && staged) {
            sts128(at0, v[0], v[1], v[2], v[3]);
            sts128(at1, v[4], v[5], v[6], v[7]);
          } else if (w.mine) {
            uint4* dst = reinterpret_cast<uint4*>(p.D + w.at + c0);
            dst[0] = make_uint4(v[0], v[1], v[2], v[3]);
            if (left > 8) dst[1] = make_uint4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      give_back();
      if constexpr (TMA_OUT > 0) {
        if (staged && w.any) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (w.row0 + 16 * h < p.rows) tma_store_2d(&map_d, buffers + h * 2048u, w.col0, w.row0 + 16 * h, store_policy);
            bulk_commit();
          }
        }
      }
      return true;
    };

    // A tile whose accumulator the next products wait for (the 256 x 256 pairs): everything into registers as raw fp32,
    // the accumulator handed back, then the same steps beside the next tile's products.
    auto pass_tile = [&](int t) {
      const Part w = part_of(t);
      const bool by_tma = whole(w);
      if constexpr (TMA_OUT > 0) {
        // The residual (dense products only, which are always stored by the TMA) comes into the staging buffer half of the
        // rows at a time; row-strided loads of it took 8192 x 8192 x 8192 from 199 to 277 us.
        if (w.any && p.residual && lane == 0) {
          bulk_wait_read<0>();  // the stores of the last tile have read the buffer
          mbar_expect_tx(res_bar, 2048u);
          tma_load_2d<1>(staging, &map_r, w.col0, w.row0, res_bar);
          tma_prefetch_2d(&map_r, w.col0, w.row0 + 16);
        }
      }
      if (!warp_wait(acc_full_bar(acc), acc_phase, 4u)) return false;
      tc_fence_after();
      uint32_t v[kCols];
      if (w.any) {
        const uint32_t acc_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * MMAS * BN);
#pragma unroll
        for (int c0 = 0; c0 < kCols; c0 += 32)
          tmem_ld_32x32(acc_tmem + (MODE == kGated ? part * 32 + c0 / 32 * (BN / 2) : part * kCols + c0),
                        *reinterpret_cast<uint32_t(*)[32]>(v + c0));
        tmem_ld_wait();
      }
      give_back();
      if (!w.any) return true;
      if constexpr (MODE == kGated) {
        if (w.mine) {
          const float gs = __ldg(p.gs + w.tile.group);
          const int col = w.tile.tn * (BN / 2) + part * 32;
          uint32_t low, high;
          uint2 first, second;
          if (p.fp16) {
            gated_block<F16Tag, false>(v, v + 32, w.alpha, gs, low, first);
            gated_block<F16Tag, false>(v + 16, v + 48, w.alpha, gs, high, second);
          } else {
            gated_block<BF16Tag, false>(v, v + 32, w.alpha, gs, low, first);
            gated_block<BF16Tag, false>(v + 16, v + 48, w.alpha, gs, high, second);
          }
          *reinterpret_cast<uint16_t*>(p.sf_out + gated_sf_offset(sf_row_of(w), col, p.N / 2)) =
              static_cast<uint16_t>(low | high << 8);
          *reinterpret_cast<uint4*>(p.out4 + static_cast<int64_t>(w.row) * (p.N / 4) + col / 2) =
              make_uint4(first.x, first.y, second.x, second.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kCols; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * w.alpha);
        if (w.bias) {
          if (p.fp16) add_bias<F16Tag, kCols>(w.bias, p.N - w.col0, v);
          else add_bias<BF16Tag, kCols>(w.bias, p.N - w.col0, v);
        }
        if (p.act != B2_ACT_NONE) activate<kCols>(p.act, v);
        if constexpr (TMA_OUT > 0) {
          if (p.residual) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h == 1 && lane == 0) {
                bulk_wait_read<0>();  // the first half's store has read the buffer
                mbar_expect_tx(res_bar, 2048u);
                tma_load_2d<1>(staging, &map_r, w.col0, w.row0 + 16, res_bar);
              }
              if (!warp_wait(res_bar, res_phase, 6u)) return false;
              res_phase ^= 1u;
              if ((lane >> 4) == h) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const uint32_t at_j = staging + (lane & 15) * 128u + ((static_cast<uint32_t>(j) ^ (lane & 7u)) * 16u);
                  uint32_t* o = v + 8 * j;
                  if (p.fp16) {
                    add8<F16Tag>(lds128_vec(at_j), o);
                    pack<F16Tag, 8>(o);
                  } else {
                    add8<BF16Tag>(lds128_vec(at_j), o);
                    pack<BF16Tag, 8>(o);
                  }
                  sts128(at_j, o[0], o[1], o[2], o[3]);
                }
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (w.row0 + 16 * h < p.rows) tma_store_2d(&map_d, staging, w.col0, w.row0 + 16 * h, store_policy);
                bulk_commit();
              }
            }
            return true;
          }
        }
        if (p.fp16) pack<F16Tag, kCols>(v);
        else pack<BF16Tag, kCols>(v);
        if (TMA_OUT > 0 && by_tma) {
          if constexpr (TMA_OUT > 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // 16 rows at a time
              if (lane == 0) bulk_wait_read<0>();  // the store that used the buffer last has read it
              __syncwarp();
              if ((lane >> 4) == h) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  sts128(staging + (lane & 15) * 128u + ((static_cast<uint32_t>(j) ^ (lane & 7u)) * 16u), v[4 * j], v[4 * j + 1],
                         v[4 * j + 2], v[4 * j + 3]);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (w.row0 + 16 * h < p.rows) tma_store_2d(&map_d, staging, w.col0, w.row0 + 16 * h, store_policy);
                bulk_commit();
              }
            }
          }
        } else if (w.mine) {
          uint4* dst = reinterpret_cast<uint4*>(p.D + w.at);
#pragma unroll
          for (int j = 0; j < kCols / 8; ++j)
            if (w.col0 + 8 * j < p.N) dst[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      }
      return true;
    };

    int t = unit;
    bool alive = true;
    if constexpr (!kAlwaysHold)
      for (; alive && t + num_units < num_tiles; t += num_units) alive = pass_tile(t);
    for (; alive && t < num_tiles; t += num_units) alive = hold_tile(t);
    if constexpr (TMA_OUT > 0) {
      if (lane == 0) bulk_wait_read<0>();  // every store has left shared memory; the end of the grid waits for the writes
    }
  }

  // ---- teardown: nobody leaves while a peer may still signal into this CTA ----
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // give copies that may still be in flight time to land before shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == kGWarpMma) {
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, kTmemCols);
  }
}

// ---- host ----------------------------------------------------------------------------------------
struct GroupedCall {
  const void *A, *B, *SFA, *SFB;
  int sfa_tiles;  // 128-row tiles of A's scale buffer
  int K;
  GroupedParams p;
  const char* who;
};

// One 16-row x 64-column store box of the 16-bit [rows, N] output, 128-byte swizzled in shared memory.
int encode_store_map(CUtensorMap* map, void* base, int rows, int N) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(N) * 2};
  const cuuint32_t box[2] = {64, 16};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base, dims, strides, box, elem,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(output) failed with %d", static_cast<int>(r));
    return B2_ERR_CUDA;
  }
  return B2_OK;
}

template <Mode MODE, int CG, int BN, int STAGES, int TMA_OUT, int AM, int MMAS, int NACC, int SETS = 2, int PARTS = 2>
int launch_grouped(const GroupedCall& c, cudaStream_t stream) {
  using L = GroupedLayout<MODE, CG, BN, STAGES, TMA_OUT, AM>;
  constexpr int kBM = AM * CG;
  auto kernel = nvfp4_grouped_gemm_kernel<MODE, CG, BN, STAGES, TMA_OUT, AM, MMAS, NACC, SETS, PARTS>;
  GroupedParams p = c.p;
  CUtensorMap map_a, map_b, map_sfa, map_sfb, map_d = {}, map_r = {};
  if (int rc = encode_operand_map(&map_a, c.A, p.rows, c.K, AM)) return rc;
  if (int rc = encode_operand_map(&map_b, c.B, p.groups * p.N, c.K, MODE == kGated ? BN / 2 : L::kBRows)) return rc;
  if (int rc = encode_scale_map(&map_sfa, c.SFA, c.sfa_tiles * 128, c.K, 1)) return rc;
  if (int rc = encode_scale_map(&map_sfb, c.SFB, p.groups * ((p.N + 127) / 128) * 128, c.K, MODE == kGated ? 1 : L::kChunks))
    return rc;
  if (TMA_OUT > 0) {
    if (int rc = encode_store_map(&map_d, p.D, p.rows, p.N)) return rc;
    if (p.residual)
      if (int rc = encode_store_map(&map_r, const_cast<uint16_t*>(p.residual), p.rows, p.N)) return rc;
  }
  p.k_slabs = (c.K + kBlockK - 1) / kBlockK;
  p.tiles_m = (p.rows + kBM - 1) / kBM;
  p.tiles_n = (p.N + BN - 1) / BN;  // gated: BN / 2 gates and BN / 2 ups a tile, the same number
  p.rcp_tiles_n = 1.0f / static_cast<float>(p.tiles_n);
  p.group_n = 8;
  const int sms = device_sm_count();
  if (sms <= 0) return B2_ERR_CUDA;
  // The most row tiles that the groups can have; for one group that is their number.
  const int64_t tiles_m = MODE != kDense ? p.rows / kBM + static_cast<int64_t>(p.groups < p.rows ? p.groups : p.rows)
                                  : p.tiles_m;
  const int64_t tiles = tiles_m * p.tiles_n;
  if (tiles > 0x3fffffff) {
    set_error("%s: %lld tiles exceed the tile list's range", c.who, static_cast<long long>(tiles));
    return B2_ERR_INVALID_ARGUMENT;
  }
  // Persistent CTAs (pairs): of a dense product as many as finish its tiles in the fewest rounds; groups may have fewer
  // tiles than `tiles`, so all that fit (with the dense rule 16384 rows of 32 groups took 13 rounds for 12).
  const int64_t rounds = (tiles + sms / CG - 1) / (sms / CG);
  const int units = static_cast<int>(MODE == kDense ? (tiles + rounds - 1) / rounds : std::min<int64_t>(tiles, sms / CG));

  {
    static std::atomic<bool> configured[64] = {};  // per instantiation; setting it twice does no harm
    int dev = 0;
    B2_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      B2_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAll));
      if (PARTS == 4) {
        // setmaxnreg hands out what the block was launched with: with fewer registers a warpgroup would wait for good.
        cudaFuncAttributes attributes;
        B2_CUDA_TRY(cudaFuncGetAttributes(&attributes, kernel));
        if (attributes.numRegs != kRegsLaunch) {
          set_error("%s: kernel built with %d registers a thread, %d expected", c.who, attributes.numRegs, kRegsLaunch);
          return B2_ERR_CUDA;
        }
      }
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * CG);
  cfg.blockDim = dim3(group_threads(SETS, PARTS));
  cfg.dynamicSmemBytes = L::kAll;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (CG == 2) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 2;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
  ++cfg.numAttrs;
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, map_sfa, map_sfb, map_d, map_r, p));
  return B2_OK;
}

// Status words of these launches: part of the library image, so that no call allocates.
static __device__ uint32_t g_grouped_status[64];

int grouped_status_words(uint32_t** out) {
  static std::atomic<uint32_t*> cache[64] = {};
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) {
    set_error("device ordinal %d out of range", dev);
    return B2_ERR_CUDA;
  }
  uint32_t* words = cache[dev].load(std::memory_order_acquire);
  if (!words) {
    void* ptr = nullptr;
    B2_CUDA_TRY(cudaGetSymbolAddress(&ptr, g_grouped_status));
    words = static_cast<uint32_t*>(ptr);
    cache[dev].store(words, std::memory_order_release);
  }
  *out = words;
  return B2_OK;
}

std::atomic<int> g_grouped_variant{-1};  // test hook: -1 = automatic

// The kernel for `rows` rows in `groups` groups (numbering of b2_nvfp4_grouped_gemm_set_variant).  Times on B200, back
// to back launches from a CUDA graph, us:
//   dense     32 x 64, 2 MMA warps   all of N in one wave of 64-wide tiles: 16 x 8192 x 8192 10.2 (32 x 128: 11.4)
//             32 x 128               more: 16 x 28672 x 8192 24.4 (32 x 64: 31.8)
//             128 x 64, 2 MMA warps  one wave of them: 1024^3 4.3 (128 x 128: 5.1, 256 x 128: 5.3), 200 x 4096 x 4096 6.6 (8.1, 7.2)
//             128 x 128              more columns, at most 128 rows: 64 x 28672 x 8192 27.2 (256 x 256: 31.2), or K up to 2048
//                                    and one wave: 1000 x 2048 x 2048 6.1 (256 x 128: 6.7; at K = 4096 both 8.2)
//             256 x 128              one wave of them: 256 x 8192 x 8192 11.1 (256 x 256: 15.2, 128 x 128: 12.7)
//             256 x 256              the rest: 2048 x 4096 x 4096 18.7 (256 x 128: 19.7)
//   grouped   32 x 128               mean of 16 rows: 1024 rows of 64, N=2048, K=4096 55.3 (128 x 128: 56.1); 8 rows,
//                                    N=4096, K=2048 11.1 (14.3)
//             128 x 128              mean of 64 rows: 4096 of 64, N=K=2048 36.5 (256 x 256: 39.3), or about one wave of
//                                    them: 777 of 7, N=1352, K=1088 7.4 (256 x 128: 8.6)
//             256 x 128              at most two waves of 256 x 256: 1024 of 8, N=K=2048 10.2 (256 x 256: 11.1, 128 x 128: 11.1)
//             256 x 256              the rest: 16384 of 32, N=2816, K=2048 65.1 (256 x 128: 73.1)
int choose_grouped_variant(int rows, int groups, bool grouped, int N, int K, int sms) {
  const int64_t n64 = (N + 63) / 64, n128 = (N + 127) / 128, n256 = (N + 255) / 256;
  if (!grouped) {
    const int64_t m128 = (rows + 127) / 128, m256 = (rows + 255) / 256;
    if (rows <= 32) return n64 <= sms ? 0 : 1;
    if (m128 * n64 <= sms) return 2;
    if (rows <= 128 || (K <= 2048 && m128 * n128 <= sms)) return 3;
    return m256 * n128 <= sms / 2 ? 5 : 4;
  }
  // The groups' sizes are known on the device alone: a group's last tile is taken to be half full.
  const int64_t mean = (static_cast<int64_t>(rows) + groups - 1) / groups;
  if (mean <= 16) return 1;
  if (mean <= 64 || (2 * (rows / 128) + groups) * n128 <= 2 * sms) return 3;
  return (2 * (rows / 256) + groups) * n256 <= 2 * sms ? 5 : 4;
}

// The two-MMA-warp kernels are for one tile per CTA, which only a dense product knows to have.  Gated, a stage of the
// 128 x 128 tiles holds one more scale chunk (five stages for six), and pairs take 256 columns: 128 gates, 128 ups.
int run_dense(int variant, const GroupedCall& c, cudaStream_t s) {
  switch (variant) {
    case 0: return launch_grouped<kDense, 1, 64, 12, 0, 32, 2, 1>(c, s);
    case 1: return launch_grouped<kDense, 1, 128, 8, 0, 32, 1, 2>(c, s);
    case 2: return launch_grouped<kDense, 1, 64, 8, 0, 128, 2, 1>(c, s);
    case 3: return launch_grouped<kDense, 1, 128, 5, 1, 128, 1, 2>(c, s);
    case 4: return launch_grouped<kDense, 2, 256, 5, 1, 128, 1, 1, 1, 4>(c, s);
    default: return launch_grouped<kDense, 2, 128, 6, 1, 128, 1, 2>(c, s);
  }
}
int run_groups(int variant, const GroupedCall& c, cudaStream_t s) {
  switch (variant) {
    case 0:
    case 1:
      // Of a 32-row tile only the epilogue warps of the first lane quarter have rows.  Where a tile has few slabs they are
      // what it waits for: twice as many parts, with half of the columns each (40 groups of one row, N = 4096: K = 512
      // 14.7 us for 17.8, K = 1024 18.0 for 19.7; K = 2048 34.4 for 33.6, with one set of scale warps).
      if (c.K <= 1024) return launch_grouped<kGrouped, 1, 128, 8, 0, 32, 1, 2, 1, 4>(c, s);
      return launch_grouped<kGrouped, 1, 128, 8, 0, 32, 1, 2>(c, s);
    case 2:
    case 3: return launch_grouped<kGrouped, 1, 128, 5, 1, 128, 1, 2>(c, s);
    case 4: return launch_grouped<kGrouped, 2, 256, 5, 1, 128, 1, 1, 1, 4>(c, s);
    default: return launch_grouped<kGrouped, 2, 128, 6, 1, 128, 1, 2>(c, s);
  }
}
int run_gated(int variant, const GroupedCall& c, cudaStream_t s) {
  switch (variant) {
    case 0:
    case 1: return launch_grouped<kGated, 1, 128, 8, 0, 32, 1, 2>(c, s);
    case 2:
    case 3: return launch_grouped<kGated, 1, 128, 5, 0, 128, 1, 2>(c, s);
    default: return launch_grouped<kGated, 2, 256, 5, 0, 128, 1, 1, 1, 4>(c, s);
  }
}

int run_grouped(const GroupedCall& c, cudaStream_t s) {
  if (!encode_tiled_fn()) {
    set_error("%s: cuTensorMapEncodeTiled is not available from this driver", c.who);
    return B2_ERR_CUDA;
  }
  const int sms = device_sm_count();
  if (sms <= 0) return B2_ERR_CUDA;
  int variant = g_grouped_variant.load(std::memory_order_relaxed);
  if (variant < 0) variant = choose_grouped_variant(c.p.rows, c.p.groups, c.p.offsets != nullptr, c.p.N, c.K, sms);
  if (c.p.out4) return run_gated(variant, c, s);
  return c.p.offsets ? run_groups(variant, c, s) : run_dense(variant, c, s);
}

// The checks that the dense and the grouped entry point share.
int check_product(const GroupedCall& c, int out_dtype) {
  const GroupedParams& p = c.p;
  if (p.rows < 0 || p.N < 1 || c.K < 1 || p.N % 8 != 0 || c.K % 64 != 0) {
    set_error("%s: %d rows, N=%d, K=%d: need rows >= 0, N %% 8 == 0, K %% 64 == 0", c.who, p.rows, p.N, c.K);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (p.groups < 1 || p.groups > kMaxGroups || static_cast<int64_t>(p.groups) * ((p.N + 127) / 128 * 128) > 0x7fffffffll ||
      p.rows > 0x7fffffff - 512) {
    set_error("%s: %d groups of N=%d with %d rows: need 1 to %d groups, groups * N and rows below 2^31", c.who,
              p.groups, p.N, p.rows, kMaxGroups);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (out_dtype != B2_DTYPE_F16 && out_dtype != B2_DTYPE_BF16) {
    set_error("%s: unsupported out_dtype %d", c.who, out_dtype);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (p.act < B2_ACT_NONE || p.act > B2_ACT_SILU) {
    set_error("%s: unknown activation %d", c.who, p.act);
    return B2_ERR_INVALID_ARGUMENT;
  }
  if (p.rows == 0) return B2_OK;
  if (!c.A || !c.B || !c.SFA || !c.SFB || !p.alpha || (!p.D && !p.out4)) {
    set_error("%s: null pointer argument", c.who);
    return B2_ERR_INVALID_ARGUMENT;
  }
  const uintptr_t all = reinterpret_cast<uintptr_t>(c.A) | reinterpret_cast<uintptr_t>(c.B) |
                        reinterpret_cast<uintptr_t>(c.SFA) | reinterpret_cast<uintptr_t>(c.SFB) |
                        reinterpret_cast<uintptr_t>(p.D) | reinterpret_cast<uintptr_t>(p.bias) |
                        reinterpret_cast<uintptr_t>(p.residual) | reinterpret_cast<uintptr_t>(p.out4);
  if ((all & 15) || ((reinterpret_cast<uintptr_t>(p.alpha) | reinterpret_cast<uintptr_t>(p.offsets)) & 3)) {
    set_error("%s: operands, scales, bias, residual and output must be 16-byte aligned, alpha and offsets 4-byte", c.who);
    return B2_ERR_INVALID_ARGUMENT;
  }
  return B2_OK;
}

}  // namespace
}  // namespace b2

extern "C" int b2_nvfp4_gemm_epilogue(const void* A, const void* B, const void* SFA, const void* SFB,
                                      const float* alpha_dev, const void* bias, const void* residual, void* D, int M,
                                      int N, int K, int out_dtype, int activation, void* stream) {
  using namespace b2;
  GroupedCall c = {};
  c.who = "b2_nvfp4_gemm_epilogue";
  c.A = A;
  c.B = B;
  c.SFA = SFA;
  c.SFB = SFB;
  c.K = K;
  c.p.alpha = alpha_dev;
  c.p.bias = static_cast<const uint16_t*>(bias);
  c.p.residual = static_cast<const uint16_t*>(residual);
  c.p.D = static_cast<uint16_t*>(D);
  c.p.rows = M;
  c.p.groups = 1;
  c.p.N = N;
  c.p.act = activation;
  c.p.fp16 = out_dtype == B2_DTYPE_F16;
  c.p.wait_budget_ns = kWaitBudgetNs;
  if (int rc = check_product(c, out_dtype)) return rc;
  if (M == 0) return B2_OK;
  c.sfa_tiles = (M + 127) / 128;
  if (int rc = grouped_status_words(&c.p.status)) return rc;
  return run_grouped(c, static_cast<cudaStream_t>(stream));
}

namespace b2 {

// The grouped products; `early` and `ids` (GroupedParams) are the routed feed-forward's (moe.cu).
int grouped_product(const void* A, const void* B, const void* SFA, const void* SFB, const float* alpha_dev,
                    const int32_t* offsets_dev, const void* bias, void* D, int rows, int groups, int N, int K,
                    int out_dtype, int activation, bool early, const int32_t* ids_dev, void* stream) {
  GroupedCall c = {};
  c.who = "b2_nvfp4_grouped_gemm";
  c.A = A;
  c.B = B;
  c.SFA = SFA;
  c.SFB = SFB;
  c.K = K;
  c.p.alpha = alpha_dev;
  c.p.offsets = offsets_dev;
  c.p.bias = static_cast<const uint16_t*>(bias);
  c.p.D = static_cast<uint16_t*>(D);
  c.p.rows = rows;
  c.p.groups = groups;
  c.p.N = N;
  c.p.act = activation;
  c.p.fp16 = out_dtype == B2_DTYPE_F16;
  c.p.early = early;
  c.p.ids = ids_dev;
  c.p.wait_budget_ns = kWaitBudgetNs;
  if (int rc = check_product(c, out_dtype)) return rc;
  if (rows == 0) return B2_OK;
  if (!offsets_dev) {
    set_error("b2_nvfp4_grouped_gemm: null pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  c.sfa_tiles = rows / 128 + groups;
  if (int rc = grouped_status_words(&c.p.status)) return rc;
  return run_grouped(c, static_cast<cudaStream_t>(stream));
}

int grouped_product_gated(const void* A, const void* B, const void* SFA, const void* SFB, const float* alpha_dev,
                          const int32_t* offsets_dev, const float* gs_dev, void* out, void* sf, int rows, int groups,
                          int inner, int K, int dtype, bool early, const int32_t* ids_dev, void* stream) {
  GroupedCall c = {};
  c.who = "b2_nvfp4_grouped_gemm_gated";
  if (inner < 128 || inner % 128 != 0 || inner > (1 << 29)) {
    set_error("b2_nvfp4_grouped_gemm_gated: inner=%d: need a positive multiple of 128", inner);
    return B2_ERR_INVALID_ARGUMENT;
  }
  c.A = A;
  c.B = B;
  c.SFA = SFA;
  c.SFB = SFB;
  c.K = K;
  c.p.alpha = alpha_dev;
  c.p.offsets = offsets_dev;
  c.p.gs = gs_dev;
  c.p.out4 = static_cast<uint8_t*>(out);
  c.p.sf_out = static_cast<uint8_t*>(sf);
  c.p.rows = rows;
  c.p.groups = groups;
  c.p.N = 2 * inner;
  c.p.act = B2_ACT_NONE;
  c.p.fp16 = dtype == B2_DTYPE_F16;
  c.p.early = early;
  c.p.ids = ids_dev;
  c.p.wait_budget_ns = kWaitBudgetNs;
  if (int rc = check_product(c, dtype)) return rc;
  if (rows == 0) return B2_OK;
  if (!offsets_dev || !gs_dev || !out || !sf || (reinterpret_cast<uintptr_t>(gs_dev) & 3) || (reinterpret_cast<uintptr_t>(sf) & 15)) {
    set_error("b2_nvfp4_grouped_gemm_gated: null or misaligned pointer argument");
    return B2_ERR_INVALID_ARGUMENT;
  }
  c.sfa_tiles = rows / 128 + groups;
  if (int rc = grouped_status_words(&c.p.status)) return rc;
  return run_grouped(c, static_cast<cudaStream_t>(stream));
}

}  // namespace b2

extern "C" int b2_nvfp4_grouped_gemm(const void* A, const void* B, const void* SFA, const void* SFB,
                                     const float* alpha_dev, const int32_t* offsets_dev, const void* bias, void* D,
                                     int rows, int groups, int N, int K, int out_dtype, int activation, void* stream) {
  return b2::grouped_product(A, B, SFA, SFB, alpha_dev, offsets_dev, bias, D, rows, groups, N, K, out_dtype, activation,
                             false, nullptr, stream);
}

extern "C" int b2_nvfp4_grouped_gemm_gated(const void* A, const void* B, const void* SFA, const void* SFB,
                                           const float* alpha_dev, const int32_t* offsets_dev, const float* gs_dev,
                                           void* out, void* sf, int rows, int groups, int inner, int K, int dtype,
                                           void* stream) {
  return b2::grouped_product_gated(A, B, SFA, SFB, alpha_dev, offsets_dev, gs_dev, out, sf, rows, groups, inner, K, dtype,
                                   false, nullptr, stream);
}

extern "C" int b2_nvfp4_grouped_gemm_set_variant(int variant) {
  if (variant < -1 || variant > 5) {
    b2::set_error("b2_nvfp4_grouped_gemm_set_variant: unknown variant %d", variant);
    return B2_ERR_INVALID_ARGUMENT;
  }
  b2::g_grouped_variant.store(variant, std::memory_order_relaxed);
  return B2_OK;
}

extern "C" int b2_nvfp4_grouped_gemm_status(void* stream) {
  using namespace b2;
  uint32_t* status = nullptr;
  if (int rc = grouped_status_words(&status)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t host[2] = {0, 0};
  B2_CUDA_TRY(cudaMemcpyAsync(host, status, sizeof(host), cudaMemcpyDeviceToHost, s));
  B2_CUDA_TRY(cudaStreamSynchronize(s));
  if (host[0] == 0) return B2_OK;
  B2_CUDA_TRY(cudaMemsetAsync(status, 0, sizeof(host), s));
  set_error("b2_nvfp4_grouped_gemm: bounded wait %u expired in CTA %u", host[0], host[1]);
  return B2_ERR_DEVICE_TIMEOUT;
}
