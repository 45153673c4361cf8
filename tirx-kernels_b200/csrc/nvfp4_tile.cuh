// Building blocks of the block-scaled NVFP4 products (nvfp4_gemm.cu, nvfp4_grouped_gemm.cu), sm_100a only:
// PTX wrappers (mbarriers, TMA, tcgen05), descriptors, the shared-memory layout of one K-slab ring, the
// bounded wait, the tile order, and the tensor maps of the operands, the scale factors and the output.
#pragma once

#include <cuda.h>

#include <mutex>

#include "common.cuh"

namespace b2 {
namespace {

constexpr int kBlockM = 128;        // rows of A per CTA (TMEM lanes)
constexpr int kBlockK = 256;        // fp4 values per stage along K = 128 bytes = one swizzle row
constexpr uint64_t kWaitBudgetNs = 1000ull * 1000ull * 1000ull;  // default budget of a wait: one second

// ---- PTX wrappers -------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint64_t globaltimer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t mapa_shared(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// Remote arrive without memory ordering: for hand-offs whose payload lives in tensor memory and
// has already been completed with tcgen05.wait, so no generic-proxy writes need publishing.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_local(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_try_wait_cluster_acquire(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;"
      " selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void fence_barrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void prefetch_tmap(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t cols) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(cols) : "memory");
  else
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(cols) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_relinquish() {
  if constexpr (CG == 1)
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  else
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
template <int CG>
__device__ __forceinline__ void tc_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                       uint32_t accumulate) {
  if constexpr (CG == 1) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p; }"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %6, 0;\n"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p; }"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
        : "memory");
  }
}
// Makes `bar` (a shared::cluster address, possibly in the peer CTA) track completion of all
// tcgen05 operations this thread issued so far.
template <int CG>
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// CTA pair: one commit that arrives on the barrier at the same shared-memory offset in both
// CTAs of the pair (a completion signal, not a load).
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// True in exactly one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{ .reg .pred P; elect.sync _|P, 0xffffffff; selp.u32 %0, 1, 0, P; }" : "=r"(pred));
  return pred != 0;
}
// One K slab from the issuing thread's side: the four MMAs and the commit that hands the stage back, with the
// poll of the barrier the thread needs NEXT issued in front of them and its result read behind them.  A poll
// takes the thread 100-200 cycles even when the barrier completed long ago (by the time the MMA thread reaches
// a stage its operands and scales have been there for ~2000 cycles), and in one instruction stream that wait
// was serial with the ~50 cycles per MMA: the thread, not the ring or the tensor pipe, set the time per slab.
// Returns whether the next barrier's phase had completed.
template <int CG>
__device__ __forceinline__ uint32_t tc_slab_and_poll_next(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                                         uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                         uint32_t sfb_step, uint32_t accumulate_first,
                                                         uint32_t commit_bar, uint32_t next_bar,
                                                         uint32_t next_parity) {
  uint32_t ok;
#define B2_MMA_(cg, d, a, b, sa, sb, pr) \
  "tcgen05.mma.cta_group::" cg ".kind::mxf4nvf4.block_scale.scale_vec::4X [" d "], " a ", " b ", %10, [" sa "], [" sb "], " pr ";\n"
  if constexpr (CG == 1) {
    asm volatile(
        "{ .reg .pred p, q, t;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%21], %22;\n"
        "setp.ne.b32 p, %19, 0;\n"
        "setp.eq.b32 t, %10, %10;\n"
        B2_MMA_("1", "%1", "%2", "%6", "%11", "%15", "p")
        B2_MMA_("1", "%1", "%3", "%7", "%12", "%16", "t")
        B2_MMA_("1", "%1", "%4", "%8", "%13", "%17", "t")
        B2_MMA_("1", "%1", "%5", "%9", "%14", "%18", "t")
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%20];\n"
        "selp.u32 %0, 1, 0, q; }"
        : "=r"(ok)
        : "r"(d_tmem), "l"(a_desc), "l"(a_desc + 2), "l"(a_desc + 4), "l"(a_desc + 6), "l"(b_desc),
          "l"(b_desc + 2), "l"(b_desc + 4), "l"(b_desc + 6), "r"(idesc), "r"(sfa), "r"(sfa + 4), "r"(sfa + 8),
          "r"(sfa + 12), "r"(sfb), "r"(sfb + sfb_step), "r"(sfb + 2 * sfb_step), "r"(sfb + 3 * sfb_step),
          "r"(accumulate_first), "r"(commit_bar), "r"(next_bar), "r"(next_parity)
        : "memory");
  } else {
    asm volatile(
        "{ .reg .pred p, q, t;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%21], %22;\n"
        "setp.ne.b32 p, %19, 0;\n"
        "setp.eq.b32 t, %10, %10;\n"
        B2_MMA_("2", "%1", "%2", "%6", "%11", "%15", "p")
        B2_MMA_("2", "%1", "%3", "%7", "%12", "%16", "t")
        B2_MMA_("2", "%1", "%4", "%8", "%13", "%17", "t")
        B2_MMA_("2", "%1", "%5", "%9", "%14", "%18", "t")
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%20], %23;\n"
        "selp.u32 %0, 1, 0, q; }"
        : "=r"(ok)
        : "r"(d_tmem), "l"(a_desc), "l"(a_desc + 2), "l"(a_desc + 4), "l"(a_desc + 6), "l"(b_desc),
          "l"(b_desc + 2), "l"(b_desc + 4), "l"(b_desc + 6), "r"(idesc), "r"(sfa), "r"(sfa + 4), "r"(sfa + 8),
          "r"(sfa + 12), "r"(sfb), "r"(sfb + sfb_step), "r"(sfb + 2 * sfb_step), "r"(sfb + 3 * sfb_step),
          "r"(accumulate_first), "r"(commit_bar), "r"(next_bar), "r"(next_parity),
          "h"(static_cast<uint16_t>(3))
        : "memory");
  }
#undef B2_MMA_
  return ok;
}
__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ---- descriptors ----------------------------------------------------------------------------
// Shared-memory matrix descriptor (sm_100 format): start address >> 4 in bits [0,14), leading
// byte offset >> 4 in [16,30), stride byte offset >> 4 in [32,46), descriptor version 1 in
// [46,48), swizzle mode in [61,64) (0 none, 2 = 128-byte).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo16, uint32_t sbo16,
                                              uint32_t layout) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lbo16 & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(sbo16 & 0x3FFFu) << 32) | (1ull << 46) | (static_cast<uint64_t>(layout) << 61);
}
// K-major operand tile stored by TMA with 128-byte swizzle: rows of 128 B, 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) { return smem_desc(addr, 1, 64, 2); }
// Instruction descriptor of kind::mxf4nvf4 with block scaling: E2M1 operands (format 1) at bits 7
// and 10, both K-major, N >> 3 at bit 17, E4M3 scales (0) at bit 23, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t instr_desc(int m, int n) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// ---- shared memory ------------------------------------------------------------------------------
// AM: rows of A the TMA writes per stage.  The MMA always reads 128 rows; with AM < 128 (M <= AM) the
// rows past AM are whatever follows in the stage, which only reaches accumulator rows nobody reads,
// and the shared memory saved buys more stages in flight.
// SFB: 128-row scale chunks of B a stage holds when they are more than BN's (0: BN's).
template <int CG, int BN, int STAGES, int TMA_OUT = 0, int AM = kBlockM, int SFB = 0>
struct SmemLayout {
  static constexpr int kBRows = BN / CG;                       // rows of B held by one CTA
  static constexpr int kChunks = BN / 128 > 0 ? BN / 128 : 1;  // 128-row scale chunks of B
  static constexpr int kABytes = AM * 128;
  static constexpr int kBBytes = kBRows * 128;
  static constexpr int kSfaBytes = 4 * 512;                    // 4 K-blocks of 64, 512 B each
  static constexpr int kSfbBytes = (SFB ? SFB : kChunks) * 4 * 512;
  static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
  static constexpr int kSfCols = 16 + 16 * kChunks;            // TMEM columns of one stage's scales
  static constexpr int kBarrierBytes = 512;
  // output staging of the TMA-store epilogue (TMA_OUT > 0): every epilogue warp owns TMA_OUT
  // sub-tiles of 32 rows x 64 bf16 columns (4 KB, 128-byte rows, 128-byte swizzle) and pushes its
  // 32 x BN/2 part of the tile through them
  static constexpr int kStagingBytes = 8 * TMA_OUT * 4096;
  static_assert(TMA_OUT == 0 || (BN / 2 / 64) % TMA_OUT == 0, "sub-tiles per warp divide its columns");
  static constexpr int kRingBytes = STAGES * kStageBytes + kStagingBytes;
  static constexpr int kTotal = kRingBytes + kBarrierBytes + 1024;  // + alignment slack
  static_assert(kStageBytes % 1024 == 0, "stages and staging stay 1024-byte aligned");
  static_assert(AM == kBlockM || (CG == 1 && kStageBytes >= kBlockM * 128), "the MMA's 128-row window stays inside the stage");
  static_assert(kTotal <= 227 * 1024, "shared memory budget");
  static_assert(BN + STAGES * kSfCols <= 512, "tensor memory budget");
  static_assert((3 * STAGES + 2) * 8 + 16 <= kBarrierBytes, "barrier area");
};

struct WaitCtx {
  uint32_t* status;
  volatile uint32_t* abort_flag;  // in shared memory
  uint64_t budget_ns;
};

// Bounded mbarrier wait.  Returns false after recording `code` when the barrier never flips or
// another role of this CTA has already given up.  The waits on data arriving from memory (codes 3
// and 5) run out after the budget, the waits downstream of them (a free stage, a drained or a
// finished accumulator) after twice the budget, so that the status word names the role that
// stalled first rather than one that only waited for it.
template <bool kClusterAcquire = false>
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, const WaitCtx& ctx,
                                              uint32_t code) {
  uint64_t started = 0;
  const uint64_t budget = (code == 3u || code == 5u) ? ctx.budget_ns : 2 * ctx.budget_ns;
  for (uint32_t i = 0;; ++i) {
    const bool ok = kClusterAcquire ? mbar_try_wait_cluster_acquire(bar, parity) : mbar_try_wait(bar, parity);
    if (ok) return true;
    if ((i & 63u) != 63u) continue;
    if (*ctx.abort_flag) return false;
    const uint64_t now = globaltimer_ns();
    if (started == 0) started = now;
    else if (now - started > budget) break;
    if (i > (1u << 26)) break;  // backstop in polls, should the timer not advance (seconds at the shortest poll)
  }
  if (atomicCAS(ctx.status, 0u, code) == 0u) ctx.status[1] = blockIdx.x;
  *ctx.abort_flag = 1u;
  return false;
}

__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int group_n, int& tm,
                                            int& tn) {
  const int per_group = group_n * tiles_m;
  const int g = t / per_group;
  const int first_n = g * group_n;
  const int width = min(group_n, tiles_n - first_n);
  const int local = t - g * per_group;
  tm = local / width;
  tn = first_n + local % width;
}

__device__ __forceinline__ void lds128(uint32_t addr, uint32_t* r) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// registers -> tensor memory: lane i of the warp writes 16 consecutive columns of TMEM lane (base + i)
__device__ __forceinline__ void tmem_st_32x32_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// The output is written once and not read again by this kernel: its lines are marked evict-first so
// that they do not push the operands, which every tile row and column re-reads, out of L2.
__device__ __forceinline__ uint64_t l2_policy_evict_first() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t smem, int x, int y, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;" ::"l"(map),
               "r"(x), "r"(y), "r"(smem), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read_all() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// ---- tensor maps (host) -------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &result) == cudaSuccess &&
        result == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

int encode_operand_map(CUtensorMap* map, const void* base, int rows, int k, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k / 2), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(k / 2)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims,
                                       strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(operand) failed with %d", static_cast<int>(r));
    return B2_ERR_CUDA;
  }
  return B2_OK;
}

// The swizzled scale buffer is [rows/128][K/64][512 bytes]; viewed as uint16 (256, K/64, rows/128),
// one load of box (256, 4, chunks) lands in shared memory as [chunk][k-block][512 B].
int encode_scale_map(CUtensorMap* map, const void* base, int rows_padded, int k, int chunks) {
  const cuuint64_t dims[3] = {256, static_cast<cuuint64_t>(k / 64), static_cast<cuuint64_t>(rows_padded / 128)};
  const cuuint64_t strides[2] = {512, static_cast<cuuint64_t>(k) * 8};
  const cuuint32_t box[3] = {256, 4, static_cast<cuuint32_t>(chunks)};
  const cuuint32_t elem[3] = {1, 1, 1};
  const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims,
                                       strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                       CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(scales) failed with %d", static_cast<int>(r));
    return B2_ERR_CUDA;
  }
  return B2_OK;
}

// One 32-row x 64-column store box of a bf16 [M, ldd] output, 128-byte swizzled in shared memory.
int encode_output_map(CUtensorMap* map, void* base, int M, int ldd) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(ldd), static_cast<cuuint64_t>(M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldd) * 2};
  const cuuint32_t box[2] = {64, 32};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, elem,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(output) failed with %d", static_cast<int>(r));
    return B2_ERR_CUDA;
  }
  return B2_OK;
}

}  // namespace
}  // namespace b2
